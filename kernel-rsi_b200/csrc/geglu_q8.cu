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
//
// What that takes: the arithmetic has to stay under the memory time, and the conversions alone would not
// (a quarter-rate instruction per value and direction).  16-bit values are worked on in pairs (f32x2);
// the largest magnitude is an integer maximum of pairs; a value is rounded to an integer by adding
// 1.5 * 2^23 (the low byte of the sum is q), and a byte becomes a float as the low byte of 2^23 + 128 + q.
#include <algorithm>

#include "common.cuh"
#include "gelu.cuh"

namespace krsi {
namespace {

using sm100::f2_add;
using sm100::f2_fma;
using sm100::f2_mul;
using sm100::f2_pack;
using sm100::f2_unpack;
using gelu::f2c;

constexpr int kGroup = 32;        // columns that share a step
constexpr int kCols = 8;          // columns of each half per thread
constexpr int kSlots = kGroup / kCols;
constexpr float kTwoC = 1.5957691216057308f;                       // 2 sqrt(2 / pi)
constexpr float kA = 0.044715f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMagic = 12582912.0f;                              // 1.5 * 2^23

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// kCols values of one half-row, as four pairs.
struct Cols {
  uint64_t v[4];
};

// s = 1 / (1 + exp(-2 z)) for a pair; exp overflows to inf for a very negative z, and s is then 0.
__device__ __forceinline__ uint64_t gate_sigmoid(uint64_t a, uint64_t a2) {
  const uint64_t x = f2_mul(a, f2_fma(a2, f2c(-kLog2e * kTwoC * kA), f2c(-kLog2e * kTwoC)));
  float x0, x1, y0, y1;
  f2_unpack(x, x0, x1);
  f2_unpack(f2_add(f2_pack(ex2_approx(x0), ex2_approx(x1)), f2c(1.0f)), y0, y1);
  return f2_pack(rcp_approx(y0), rcp_approx(y1));
}

// Up to kCols columns from p (the columns from `left` on are zero), VEC at a time: VEC divides F, so an
// access is inside the row or outside it.
template <typename T, int VEC>
__device__ __forceinline__ void load_raw(const T* p, int left, T* v) {
#pragma unroll
  for (int k = 0; k < kCols; k += VEC) {
    Pack<T, VEC> r;
    memset(&r, 0, sizeof(r));
    if (k < left) r = *reinterpret_cast<const Pack<T, VEC>*>(p + k);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[k + e] = r.v[e];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_raw(T* p, int left, const T* v) {
#pragma unroll
  for (int k = 0; k < kCols; k += VEC)
    if (k < left) {
      Pack<T, VEC> r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = v[k + e];
      *reinterpret_cast<Pack<T, VEC>*>(p + k) = r;
    }
}

// One half-row's columns of a storage type: the raw values, widened and narrowed in pairs.
template <int DT>
struct alignas(16) Raw {
  using T = typename Elem<DT>::T;
  T v[kCols];
  __device__ __forceinline__ Cols widen() const {
    Cols c;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (DT == KRSI_F32) c.v[k] = f2_pack(v[2 * k], v[2 * k + 1]);
      else c.v[k] = gelu::widen<DT == KRSI_F16>(reinterpret_cast<const uint32_t*>(v)[k]);
    }
    return c;
  }
  __device__ __forceinline__ void narrow(const Cols& c) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (DT == KRSI_F32) f2_unpack(c.v[k], v[2 * k], v[2 * k + 1]);
      else reinterpret_cast<uint32_t*>(v)[k] = gelu::narrow<DT == KRSI_F16>(c.v[k]);
    }
  }
  // The largest magnitude as fp32 bits (which order as integers: NaN above infinity above the rest).
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (DT == KRSI_F32) {
      uint32_t t = 0;
#pragma unroll
      for (int k = 0; k < kCols; ++k) t = max(t, __float_as_uint(v[k]) & 0x7fffffffu);
      return t;
    } else {
      uint32_t t = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t m = reinterpret_cast<const uint32_t*>(v)[k] & 0x7fff7fffu;
        asm("max.u16x2 %0, %0, %1;" : "+r"(t) : "r"(m));
      }
      const uint32_t h = max(t & 0xffffu, t >> 16);
      return DT == KRSI_BF16 ? h << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
    }
  }
};

// The group's largest magnitude over its 4 lanes.
__device__ __forceinline__ uint32_t group_top(uint32_t t) {
  t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
  return max(t, __shfl_xor_sync(0xffffffffu, t, 2));
}
__device__ __forceinline__ uint32_t exponent_of(uint32_t top) {
  return top >= 0x7f800000u ? 255u : max(top >> 23, 7u) - 6u;   // at least 1: a step of 2^-126
}
__device__ __forceinline__ float step_of(uint32_t e) { return __uint_as_float(e == 255u ? 0x7fffffffu : e << 23); }

template <int VEC>
__device__ __forceinline__ void store_q(int8_t* p, int left, const Cols& c, uint32_t top, uint32_t e) {
  const float inv = __uint_as_float((254u - min(e, 253u)) << 23);   // 1 / step
  uint32_t w[2];
  uint32_t y[kCols];
  if (__uint_as_float(top) * inv < 127.5f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t r = f2_fma(c.v[k], f2c(inv), f2c(kMagic));
      y[2 * k] = (uint32_t)r;
      y[2 * k + 1] = (uint32_t)(r >> 32);
    }
  } else {   // (or not finite: anything) some value may round to 128: held at 127
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float x0, x1;
      f2_unpack(f2_mul(c.v[k], f2c(inv)), x0, x1);
      y[2 * k] = __float_as_uint(fminf(fmaxf(x0, -127.f), 127.f) + kMagic);
      y[2 * k + 1] = __float_as_uint(fminf(fmaxf(x1, -127.f), 127.f) + kMagic);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = __byte_perm(__byte_perm(y[4 * h], y[4 * h + 1], 0x0040), __byte_perm(y[4 * h + 2], y[4 * h + 3], 0x0040),
                       0x5410);
  store_raw<int8_t, VEC>(p, left, reinterpret_cast<const int8_t*>(w));
}
struct alignas(8) Bytes {
  int8_t v[kCols];
};
template <int VEC>
__device__ __forceinline__ Bytes load_q(const int8_t* p, int left) {
  Bytes b;
  load_raw<int8_t, VEC>(p, left, b.v);
  return b;
}
__device__ __forceinline__ Cols dequantise(const Bytes& b, uint32_t e) {
  const uint64_t step = f2c(step_of(e));
  Cols c;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(b.v)[k / 2] ^ 0x80808080u;   // q + 128
    const uint32_t lo = __byte_perm(w, 0x4B000000u, 0x7440 | (k % 2 * 2));           // 2^23 + q + 128
    const uint32_t hi = __byte_perm(w, 0x4B000000u, 0x7440 | (k % 2 * 2 + 1));
    c.v[k] = f2_mul(f2_add((uint64_t)hi << 32 | lo, f2c(-8388736.0f)), step);
  }
  return c;
}

// One item, 8 columns of both halves of a row, per thread, in row order: many short blocks, all of whose
// loads are issued at once, keep more in flight than fewer blocks that loop over the rows
// (measured at 32,768 rows of F = 4,608 in bf16: 212 and 203 us forward and backward, against 277 and 290 with 8
// looping blocks per SM, and 228 and 261 with two items per thread).
struct Rows {
  uint32_t items, slots, mul, shift;   // slots: items per row, divided by as (umulhi(i, mul) + i) >> shift
  int F;
};
struct Place {
  uint32_t row, slot;
  int left;             // columns from the item's first to the end of the half-row; 0: no item
  int64_t at, half;     // offsets in [rows, 2F] (the gate's; the value's is F further) and in [rows, F]
  __device__ __forceinline__ Place(const Rows& r, uint32_t i) {
    row = (__umulhi(i, r.mul) + i) >> r.shift;
    slot = i - row * r.slots;
    left = i < r.items ? r.F - (int)(slot * kCols) : 0;
    half = (int64_t)row * r.F + slot * kCols;
    at = half + (int64_t)row * r.F;
  }
};

template <int DT, int VEC>
__global__ void __launch_bounds__(256)
geglu_q8_fwd_kernel(const typename Elem<DT>::T* __restrict__ u, typename Elem<DT>::T* __restrict__ out,
                    int8_t* __restrict__ q, uint8_t* __restrict__ ex, const Rows r) {
  pdl_enter();
  using T = typename Elem<DT>::T;
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  const Place p(r, i);
  Raw<DT> ra, rb, ro;
  load_raw<T, VEC>(u + p.at, p.left, ra.v);
  load_raw<T, VEC>(u + p.at + r.F, p.left, rb.v);
  const Cols a = ra.widen(), b = rb.widen();
  Cols o;
#pragma unroll
  for (int k = 0; k < 4; ++k) o.v[k] = f2_mul(f2_mul(a.v[k], gate_sigmoid(a.v[k], f2_mul(a.v[k], a.v[k]))), b.v[k]);
  ro.narrow(o);
  store_raw<T, VEC>(out + p.half, p.left, ro.v);
  if (q == nullptr) return;
  const uint32_t ta = group_top(ra.top()), tb = group_top(rb.top());   // every lane meets the shuffles
  const uint32_t ea = exponent_of(ta), eb = exponent_of(tb);
  store_q<VEC>(q + p.at, p.left, a, ta, ea);
  store_q<VEC>(q + p.at + r.F, p.left, b, tb, eb);
  if (p.left > 0 && i % kSlots == 0)   // [row][group][gate, value]
    *reinterpret_cast<uint16_t*>(ex + i / kSlots * 2) = (uint16_t)(ea | eb << 8);
}

// From the checkpoint's gate a and value b and the output's gradient g: d(gate), d(value) and, where OUT,
// the output again.  HUGE: a^2 may overflow; it is held finite, so that a slope of 0 times it is 0.
template <bool OUT, bool HUGE>
__device__ __forceinline__ void grad_cols(Cols& a, Cols& b, const Cols& g, Cols& o) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint64_t a2 = f2_mul(a.v[k], a.v[k]);
    if (HUGE) {
      float lo, hi;
      f2_unpack(a2, lo, hi);
      a2 = f2_pack(fminf(lo, 1e30f), fminf(hi, 1e30f));
    }
    const uint64_t s = gate_sigmoid(a.v[k], a2), gel = f2_mul(a.v[k], s);
    const uint64_t rest = f2_fma(s ^ 0x8000000080000000ull, gel, gel);                  // gel (1 - s)
    const uint64_t slope = f2_fma(rest, f2_fma(a2, f2c(3.0f * kA * kTwoC), f2c(kTwoC)), s);
    if (OUT) o.v[k] = f2_mul(gel, b.v[k]);
    a.v[k] = f2_mul(f2_mul(g.v[k], b.v[k]), slope);
    b.v[k] = f2_mul(g.v[k], gel);
  }
}

template <int DT, int VEC, bool OUT>
__global__ void __launch_bounds__(256)
geglu_q8_bwd_kernel(const typename Elem<DT>::T* __restrict__ g, const int8_t* __restrict__ q,
                    const uint8_t* __restrict__ ex, typename Elem<DT>::T* __restrict__ du,
                    typename Elem<DT>::T* __restrict__ out, const Rows r) {
  pdl_enter();
  using T = typename Elem<DT>::T;
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  const Place p(r, i);
  if (p.left <= 0) return;
  const Bytes qa = load_q<VEC>(q + p.at, p.left), qb = load_q<VEC>(q + p.at + r.F, p.left);
  Raw<DT> w;
  load_raw<T, VEC>(g + p.half, p.left, w.v);
  const uint32_t e = *reinterpret_cast<const uint16_t*>(ex + i / kSlots * 2);
  Cols a = dequantise(qa, e & 255u), b = dequantise(qb, e >> 8), o;
  const Cols gv = w.widen();
  // values of 2^7 2^(e - 127) and less: their squares stay below 2^127 up to e = 183
  if (DT == KRSI_F16 || (e & 255u) <= 183u) grad_cols<OUT, false>(a, b, gv, o);
  else grad_cols<OUT, true>(a, b, gv, o);
  w.narrow(a);
  store_raw<T, VEC>(du + p.at, p.left, w.v);
  w.narrow(b);
  store_raw<T, VEC>(du + p.at + r.F, p.left, w.v);
  if (OUT) {
    w.narrow(o);
    store_raw<T, VEC>(out + p.half, p.left, w.v);
  }
}

inline uint32_t slots_of(int64_t F) { return (uint32_t)((F + kGroup - 1) / kGroup * kSlots); }
// A launch takes at most this many rows, so that its items fit 31 bits.
inline int64_t rows_per_launch(int64_t F) { return ((int64_t)1 << 31) / slots_of(F) - 1; }
inline Rows rows_of(int64_t rows, int64_t F) {
  Rows r;
  r.slots = slots_of(F);
  r.items = (uint32_t)rows * r.slots;
  r.F = (int)F;
  r.shift = 0;
  while (((uint64_t)1 << r.shift) < r.slots) ++r.shift;
  r.mul = (uint32_t)((((uint64_t)1 << (32 + r.shift)) + r.slots - 1) / r.slots - ((uint64_t)1 << 32));
  return r;
}

template <int DT, int VEC>
int fwd(const void* u, void* out, void* q, void* ex, int64_t rows, int64_t F, cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  for (int64_t r0 = 0; r0 < rows; r0 += rows_per_launch(F)) {
    const Rows r = rows_of(std::min(rows - r0, rows_per_launch(F)), F);
    KRSI_CUDA_TRY(launch_pdl(geglu_q8_fwd_kernel<DT, VEC>, dim3((r.items + 255) / 256), dim3(256), 0, stream,
                             (const T*)u + r0 * 2 * F, (T*)out + r0 * F, q ? (int8_t*)q + r0 * 2 * F : nullptr,
                             (uint8_t*)ex + r0 * (r.slots / kSlots) * 2, r));
  }
  return KRSI_OK;
}
template <int DT, int VEC>
int bwd(const void* g, const void* q, const void* ex, void* du, void* out, int64_t rows, int64_t F,
        cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  auto kern = out ? geglu_q8_bwd_kernel<DT, VEC, true> : geglu_q8_bwd_kernel<DT, VEC, false>;
  for (int64_t r0 = 0; r0 < rows; r0 += rows_per_launch(F)) {
    const Rows r = rows_of(std::min(rows - r0, rows_per_launch(F)), F);
    KRSI_CUDA_TRY(launch_pdl(kern, dim3((r.items + 255) / 256), dim3(256), 0, stream, (const T*)g + r0 * F,
                             (const int8_t*)q + r0 * 2 * F, (const uint8_t*)ex + r0 * (r.slots / kSlots) * 2,
                             (T*)du + r0 * 2 * F, out ? (T*)out + r0 * F : nullptr, r));
  }
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
  if (bits_of(exponents) % 2 != 0) return KRSI_ERR_MISALIGNED;
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
  if (bits_of(exponents) % 2 != 0) return KRSI_ERR_MISALIGNED;
  const int es = dtype == KRSI_F32 ? 4 : 2;
  const int vec = access_cols(F, es, bits_of(g) | bits_of(du) | bits_of(out), bits_of(q));
  KRSI_Q8_DISPATCH(bwd, vec, g, q, exponents, du, out, rows, F, stream)
}
