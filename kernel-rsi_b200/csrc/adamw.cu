// adamw.cu - one AdamW step over many tensors, its states in fp32 or 8 bits, for B200:
//   g' = c g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,  t = t + 1
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// c = min(1, max_norm / (|g| + 1e-6)) with |g| the norm of all gradients together, or 1.  A norm that is not finite
// leaves everything as it is, t included.  A weight in 16 bits may have an fp32 master, which is then what is
// updated; the weight is its rounding.
//
// Launches: the sums of squares (only where max_norm is given), one block that turns them and the step into the
// factors (t lives on the device, so a captured step counts on when it is replayed), and the update.  The tensors'
// addresses travel as kernel arguments: nothing on the device has to be kept or copied for them.
//
// 8-bit states: m and r = sqrt(v) as e4m3 at a power of two for each group of 256 values, which puts the group's
// largest magnitude into [128, 256): 13 binades below it keep 3 bits of mantissa, three more lose one each.  r and not
// v, because a square takes twice the binades.  r is rounded up or down at random, right on average: it moves by far
// less than half a code a step, and rounded to nearest it would stay where it is.  So does m wherever (1 - b1) |g' - m|
// is below half a code: rounded to nearest it stops at 0.71 of a constant gradient (b1 0.9; 0.54 at 0.95), and the last
// codes of an element without gradients never go.  With KRSI_ADAMW_RANDOM_M it is rounded at random too, by other
// bits, which holds over a run of steps; without, one step's codes are the nearest ones.  The randomness is a hash of
// the element's place and t, so a step has the same bits every time.  A positive v never becomes 0, which eps alone
// would divide by.
// A group with a value that is not finite reads back as NaN.
// The moments and their codes are formed by IEEE operations in a fixed order without contraction.
#include <math.h>

#include <cuda_fp8.h>

#include "common.cuh"
#include "sm100.cuh"

namespace krsi {
namespace {

constexpr int kGroup = 256;                        // values that share the exponents of 8-bit states
constexpr int kThreads = 256;
constexpr int kGroupsPerWarp = 4;                  // at most
constexpr int kChunk = kThreads / 32 * kGroupsPerWarp * kGroup;   // values of one block, at most: 8192
constexpr int kLane = 8;                           // values of one lane
constexpr int kBlocks8 = 444;                      // 8-bit states: blocks, three an SM
constexpr int kNormBlocks = 592;                   // a fixed cap, so that the sum's order does not depend on the GPU
constexpr int kSmallCap = 24, kLargeCap = 440;     // tensors of one launch: 1.6 and 28 KB of kernel arguments

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* master;
  uint8_t* exponents;
  int64_t n;
  int first_chunk;   // chunks (8-bit states: groups) of the tensors before it in the launch
  int aligned;       // whether every pointer allows a lane's vector accesses
};

template <int CAP>
struct Table {
  Tensor t[CAP];
  int count, n_chunks;
};

// What the update takes from the device.
struct Factors {
  float clip, rate, inv_root, decay;
  uint32_t step;
  int skip;
};
constexpr size_t kFactorBytes = 256;

// The tensor that a chunk belongs to: the last one that begins at or before it.
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& tab, int chunk) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first_chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ---------------------------------------------------------------- a lane's eight values
__device__ __forceinline__ void load8(const float* p, float* o) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(o[0]), "=f"(o[1]), "=f"(o[2]), "=f"(o[3]), "=f"(o[4]), "=f"(o[5]), "=f"(o[6]), "=f"(o[7])
               : "l"(p));
}
__device__ __forceinline__ void store8(float* p, const float* o) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(o[0]), "f"(o[1]), "f"(o[2]),
               "f"(o[3]), "f"(o[4]), "f"(o[5]), "f"(o[6]), "f"(o[7])
               : "memory");
}
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t at, bool vec, int live, float* o) {
  using E = Elem<DT>;
  using T = typename E::T;
  const T* p = static_cast<const T*>(base) + at;
  if (vec) {
    if constexpr (DT == KRSI_F32) {
      load8(p, o);
    } else {
      Vec16<T> u;
      *reinterpret_cast<uint4*>(&u) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
      for (int e = 0; e < kLane; ++e) o[e] = E::load(u.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kLane; ++e) o[e] = e < live ? E::load(p[e]) : 0.f;
  }
}
template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t at, bool vec, int live, const float* o) {
  using E = Elem<DT>;
  using T = typename E::T;
  T* p = static_cast<T*>(base) + at;
  if (vec) {
    if constexpr (DT == KRSI_F32) {
      store8(p, o);
    } else {
      Vec16<T> u;
#pragma unroll
      for (int e = 0; e < kLane; ++e) u.v[e] = E::store(o[e]);
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kLane; ++e)
      if (e < live) p[e] = E::store(o[e]);
  }
}

// ---------------------------------------------------------------- codes
// 2^(byte - 127), NaN for the mark of a group that is not finite.
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fffffffu : byte << 23);
}
// 2^(127 - byte), byte at most 253
__device__ __forceinline__ float inverse_scale_of(uint32_t byte) {
  return __uint_as_float((254 - byte) << 23);
}
// 16 random bits for each of a pair of places (low half: the even one).
__device__ __forceinline__ uint32_t dither(uint32_t pair, uint32_t step) {
  uint32_t h = pair * 0x9E3779B1u + step * 0x632BE5ABu;
  h = (h ^ (h >> 16)) * 0x21F0AAADu;
  h = (h ^ (h >> 15)) * 0x735A2D97u;
  return h ^ (h >> 15);
}
// As many for m, independent of those that round r: counted over all h, each combination of the first six bits of a half
// of either is equally frequent, to 0.2%.
__device__ __forceinline__ uint32_t dither_m(uint32_t h) {
  h *= 0x2C1B3C6Du;
  return h ^ (h >> 16);
}

// ---------------------------------------------------------------- kernels
template <int GT, int CAP>
__global__ void __launch_bounds__(kThreads)
adamw_norm_kernel(const __grid_constant__ Table<CAP> tab, double* __restrict__ partial) {
  pdl_enter();
  __shared__ double red[kThreads / 32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  double sum = 0.0;
  for (int chunk = blockIdx.x; chunk < tab.n_chunks; chunk += gridDim.x) {
    const Tensor& t = tab.t[tensor_of(tab, chunk)];
    const int64_t base = (int64_t)(chunk - t.first_chunk) * kChunk + warp * (kGroupsPerWarp * kGroup) + lane * kLane;
    float g[kGroupsPerWarp][kLane];
#pragma unroll
    for (int j = 0; j < kGroupsPerWarp; ++j) {
      const int64_t at = base + j * kGroup, left = t.n - at;
      load8<GT>(t.g, at, t.aligned && left >= kLane, left > kLane ? kLane : (int)(left < 0 ? 0 : left), g[j]);
    }
    // 64 bits throughout: the factor is then the same fp32 number whatever the order (8-bit codes that lie next to a
    // border would follow its last bit)
#pragma unroll
    for (int j = 0; j < kGroupsPerWarp; ++j)
#pragma unroll
      for (int e = 0; e < kLane; ++e) sum = fma((double)g[j][e], (double)g[j][e], sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) total += red[i];
    partial[blockIdx.x] = total;
  }
}

struct FactorArgs {
  const double* partial;
  int n_partials;
  float* norm;           // or null
  int64_t* step;
  const float* lr_dev;   // or null: lr
  double lr, log_beta1, log_beta2, decay;
  float max_norm;        // 0: none
};

__global__ void __launch_bounds__(256)
adamw_factors_kernel(const FactorArgs a, Factors* __restrict__ out) {
  pdl_enter();
  __shared__ double red[8];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  double sum = 0.0;
  for (int i = threadIdx.x; i < a.n_partials; i += 256) sum += a.partial[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  if (warp != 0) return;
  Factors f{1.f, 0.f, 0.f, 0.f, 0u, 0};
  if (a.max_norm > 0.f) {
    double total = 0.0;
    for (int i = 0; i < 8; ++i) total += red[i];
    const float norm = (float)sqrt(total);
    if (lane == 0) *a.norm = norm;
    f.clip = fminf(__fdiv_rn(a.max_norm, __fadd_rn(norm, 1e-6f)), 1.f);
    f.skip = !isfinite(norm);
  }
  if (!f.skip) {
    const int64_t t = *a.step + 1;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    // 1 - beta^t, of beta1 in the even lanes and of beta2 in the odd ones
    const double bias = -expm1((double)t * (lane % 2 == 0 ? a.log_beta1 : a.log_beta2));
    const double bias2 = __shfl_sync(0xffffffffu, bias, 1);
    __syncwarp();   // every lane has read the step
    if (lane == 0) *a.step = t;
    f.rate = (float)(lr / bias);
    f.inv_root = (float)(1.0 / sqrt(bias2));
    f.decay = (float)(1.0 - lr * a.decay);
    f.step = (uint32_t)t;
  }
  if (lane == 0) *out = f;
}

struct Rates {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps;
};
// Each twice, for f32x2 operations on kernel arguments.  `one` is there for sums of products that are to be rounded
// before they are added: a paired multiplication and addition, .rn or not, come out of the assembler as one fma; the
// addition as an fma by a 1 that it does not know cannot be joined to either product.
struct RatePairs {
  float2 beta1, one_minus_beta1, beta2, one_minus_beta2, eps, one{1.f, 1.f};
  explicit RatePairs(const Rates& r)
      : beta1{r.beta1, r.beta1}, one_minus_beta1{r.one_minus_beta1, r.one_minus_beta1}, beta2{r.beta2, r.beta2},
        one_minus_beta2{r.one_minus_beta2, r.one_minus_beta2}, eps{r.eps, r.eps} {}
};

template <int PT, int GT, bool MASTER, int CAP>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(const __grid_constant__ Table<CAP> tab, const Rates c, const int groups,
             const Factors* __restrict__ factors) {
  const int lane = threadIdx.x % 32;
  const Tensor& t = tab.t[tensor_of(tab, blockIdx.x)];
  const int64_t base = ((int64_t)(blockIdx.x - t.first_chunk) * (kThreads / 32) + threadIdx.x / 32) * groups * kGroup;
  const int64_t n = t.n;
  float p[kLane], g[kLane], m[kLane], v[kLane];
  auto load = [&](int j) {
    const int64_t at = base + j * kGroup + lane * kLane, left = n - at;
    const bool vec = t.aligned && left >= kLane;
    const int live = left > kLane ? kLane : (int)(left < 0 ? 0 : left);
    if constexpr (MASTER) load8<KRSI_F32>(t.master, at, vec, live, p);
    else load8<PT>(t.p, at, vec, live, p);
    load8<GT>(t.g, at, vec, live, g);
    load8<KRSI_F32>(t.m, at, vec, live, m);
    load8<KRSI_F32>(t.v, at, vec, live, v);
  };
  pdl_enter();
  load(0);   // (beside the factors: 32M values in 106 us, after them in 117)
  const Factors f = *factors;
  if (f.skip) return;
#pragma unroll 1
  for (int j = 0; j < groups; ++j) {
    const int64_t at = base + j * kGroup + lane * kLane, left = n - at;
    if (left <= 0) return;
    const bool vec = t.aligned && left >= kLane;
    const int live = left > kLane ? kLane : (int)left;
    if (j > 0) load(j);
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      const float ge = __fmul_rn(g[e], f.clip);
      m[e] = __fadd_rn(__fmul_rn(m[e], c.beta1), __fmul_rn(ge, c.one_minus_beta1));
      v[e] = __fadd_rn(__fmul_rn(v[e], c.beta2), __fmul_rn(__fmul_rn(ge, ge), c.one_minus_beta2));
      // (the quotient to 2 units of its last place, of a move that is some thousandth of p)
      p[e] = p[e] * f.decay - f.rate * __fdividef(m[e], fmaf(sqrtf(v[e]), f.inv_root, c.eps));
    }
    if constexpr (MASTER) store8<KRSI_F32>(t.master, at, vec, live, p);
    store8<PT>(t.p, at, vec, live, p);
    store8<KRSI_F32>(t.m, at, vec, live, m);
    store8<KRSI_F32>(t.v, at, vec, live, v);
  }
}

// ---------------------------------------------------------------- 8-bit states
// At 10 bytes a bf16 weight the memory leaves some 50 issued instructions to each, so the arithmetic is what has to be
// short: pairs of fp32 (f32x2) where IEEE operations are wanted, one SFU instruction each for the root and the
// quotient, and the next group's loads in flight meanwhile. The codes nevertheless follow the correctly rounded root:
// where the SFU's could round the other way (once in 2^17 values) the lane takes __fsqrt_rn.

// A lane's eight values as they are in memory.
template <int DT>
struct Raw8 {
  static constexpr int W = DT == KRSI_F32 ? 8 : 4;
  uint32_t w[W];
  __device__ __forceinline__ uint64_t pair(int k) const {   // values 2k and 2k + 1 in fp32
    if constexpr (DT == KRSI_F32) return sm100::f2_pack(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    else if constexpr (DT == KRSI_BF16)
      return sm100::f2_pack(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
    else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      return sm100::f2_pack(f.x, f.y);
    }
  }
};
template <int DT>
__device__ __forceinline__ void load_raw(Raw8<DT>& r, const void* base, int64_t at, bool vec, int live) {
  using T = typename Elem<DT>::T;
  const T* p = static_cast<const T*>(base) + at;
  if (vec) {
    if constexpr (DT == KRSI_F32) {
      float o[8];
      load8(reinterpret_cast<const float*>(p), o);
#pragma unroll
      for (int k = 0; k < 8; ++k) r.w[k] = __float_as_uint(o[k]);
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      r.w[0] = u.x; r.w[1] = u.y; r.w[2] = u.z; r.w[3] = u.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < Raw8<DT>::W; ++k) r.w[k] = 0;
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      if (e >= live) continue;
      if constexpr (DT == KRSI_F32) r.w[e] = __float_as_uint(p[e]);
      else r.w[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e % 2));
    }
  }
}
__device__ __forceinline__ uint2 load_codes(const void* base, int64_t at, bool vec, int live) {
  const uint8_t* p = static_cast<const uint8_t*>(base) + at;
  if (vec) return *reinterpret_cast<const uint2*>(p);
  uint32_t u[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < kLane; ++e)
    if (e < live) u[e / 4] |= (uint32_t)p[e] << (8 * (e % 4));
  return make_uint2(u[0], u[1]);
}
__device__ __forceinline__ uint2 pack_codes(const float* o) {
  uint32_t u[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(o[4 * k], o[4 * k + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(o[4 * k + 2], o[4 * k + 3]), __NV_SATFINITE, __NV_E4M3);
    u[k] = __byte_perm(lo, hi, 0x5410);
  }
  return make_uint2(u[0], u[1]);
}
__device__ __forceinline__ void store_codes(void* base, int64_t at, bool vec, int live, uint2 u) {
  uint8_t* p = static_cast<uint8_t*>(base) + at;
  if (vec) {
    *reinterpret_cast<uint2*>(p) = u;
  } else {
#pragma unroll
    for (int e = 0; e < kLane; ++e)
      if (e < live) p[e] = (uint8_t)((e < 4 ? u.x : u.y) >> (8 * (e % 4)));
  }
}
// Codes 2k and 2k + 1 as fp32.
__device__ __forceinline__ uint64_t decode_pair(uint2 u, int k) {
  const uint32_t w = k < 2 ? u.x : u.y;
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(k % 2 ? w >> 16 : w & 0xffff), __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return sm100::f2_pack(f.x, f.y);
}
__device__ __forceinline__ float sqrt_sfu(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest of three magnitudes; NaN if one is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max8_abs(const float* x) {
  return max3_abs(max3_abs(x[0], x[1], x[2]), max3_abs(x[3], x[4], x[5]), max3_abs(x[6], x[7], x[7]));
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

constexpr float kLift = 0.015625f;       // 2^-6: codes below are subnormal, 2^-9 apart
constexpr float kLeast = 0.001953125f;   // 2^-9, the least positive code

// Scaled roots x >= 2^-6 to codes: up with the probability of the bits below the code's last one.  They and the random
// bits (below fp32's 20th) carry into it; half a code less, the conversion's rounding to nearest then cuts them off.
// False if one of them came within 8 units of x's last place of rounding differently.
__device__ __forceinline__ bool round_roots(const float* x, const uint32_t* h, float* code) {
  int nearest = 0x7fffffff;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t lo = __float_as_uint(x[2 * k]) + ((h[k] << 4) & 0xffff0u) + (8u - 0x80000u);
    const uint32_t hi = __float_as_uint(x[2 * k + 1]) + ((h[k] >> 16) << 4) + (8u - 0x80000u);
    nearest = min(nearest, min((int)(lo << 12), (int)(hi << 12)));   // (half a code less: the sign bit)
    code[2 * k] = __uint_as_float(lo);
    code[2 * k + 1] = __uint_as_float(hi);
  }
  return nearest >= (int)0x80010000;
}
// The same for any v, from its correctly rounded root: 2^-6 more puts roots below 2^-6 where fp32's 20th bit is worth
// 2^-9; a positive one gives at least the least code.
__device__ __forceinline__ float round_root(float v, float inverse_scale, uint32_t random16) {
  const float x = __fmul_rn(__fsqrt_rn(v), inverse_scale);
  const float lift = x < kLift ? kLift : 0.f;
  const uint32_t up = (__float_as_uint(__fadd_rn(x, lift)) + (random16 << 4)) & 0xfff00000u;
  return x > 0.f ? fmaxf(__fadd_rn(__uint_as_float(up), -lift), kLeast) : 0.f;
}

// Four scaled m, |x| < 2^8, to codes, up in magnitude with the probability of what lies below the code's last bit.  2^-120
// takes e4m3's least normal number, 2^-6, to fp32's: from there on the codes are fp32's leading bits, those of subnormal
// numbers and of zero too, so the random bits are added below them and the rest is cut off.
// (632M weights, a tenth without gradients: 1171 us, to nearest 1119; by conversions, with another way for lanes that have a
// value below 2^-6, 1466.)
__device__ __forceinline__ uint32_t random_codes(uint64_t x01, uint64_t x23, uint32_t h01, uint32_t h23) {
  using namespace sm100;
  const uint64_t down = f2_pack(0x1p-120f, 0x1p-120f);
  float f[4];
  f2_unpack(f2_mul(x01, down), f[0], f[1]);
  f2_unpack(f2_mul(x23, down), f[2], f[3]);
  uint32_t b[4], up[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    b[e] = __float_as_uint(f[e]);
    // the code's seven bits to the top byte, the random 16 to those below (byte 0 stays 0)
    up[e] = (b[e] << 4) + __byte_perm(e < 2 ? h01 : h23, 0, e % 2 ? 0x4324 : 0x4104);
  }
  auto top_bytes = [](const uint32_t* u) {
    return __byte_perm(__byte_perm(u[0], u[1], 0x0073), __byte_perm(u[2], u[3], 0x0073), 0x5410);
  };
  return top_bytes(up) | (top_bytes(b) & 0x80808080u);
}

// A lane's part of a group: as read, and the results.
template <int WT, int GT>
struct Lane8 {
  Raw8<WT> p;
  Raw8<GT> g;
  uint2 m, r;
  uint32_t ex;   // both exponents
};
struct Done8 {
  float p[kLane];
  uint2 m, r;
  uint32_t ex;
};
// Called by whole warps.  pair: the place of the lane's first value, halved.
template <int WT, int GT, bool RANDOM_M>
__device__ __forceinline__ void update8(const Lane8<WT, GT>& in, const RatePairs& c, const Factors& f, uint32_t pair,
                                        Done8& out) {
  using namespace sm100;
  const auto pair_of = [](const float2& x) { return *reinterpret_cast<const uint64_t*>(&x); };
  const auto twice = [](float x) { return f2_pack(x, x); };
  uint64_t m[4], v[4];
  {
    const uint64_t sm = twice(scale_of(in.ex & 0xff)), sr = twice(scale_of(in.ex >> 8)), clip = twice(f.clip);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t g = f2_mul(in.g.pair(k), clip);
      m[k] = f2_fma(f2_mul(f2_mul(decode_pair(in.m, k), sm), pair_of(c.beta1)), pair_of(c.one),
                    f2_mul(g, pair_of(c.one_minus_beta1)));
      const uint64_t r = f2_mul(decode_pair(in.r, k), sr);
      v[k] = f2_fma(f2_mul(f2_mul(r, r), pair_of(c.beta2)), pair_of(c.one),
                    f2_mul(f2_mul(g, g), pair_of(c.one_minus_beta2)));
    }
  }
  float mf[kLane], vf[kLane];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f2_unpack(m[k], mf[2 * k], mf[2 * k + 1]);
    f2_unpack(v[k], vf[2 * k], vf[2 * k + 1]);
  }
  const int field_m = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(max8_abs(mf))) >> 23);
  const int field_v = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(max8_abs(vf))) >> 23);
  // the group's largest magnitude 2^k f, 1 <= f < 2, becomes 2^7 f (one that is not finite marks the group; its own
  // weights are still updated one by one)
  const uint32_t em = field_m >= 255 ? 127u : (uint32_t)max(field_m - 7, 1);
  const uint32_t er = field_v >= 255 ? 127u : (uint32_t)(((field_v - 127) >> 1) + 120);
  out.ex = (field_m >= 255 ? 255u : em) | ((field_v >= 255 ? 255u : er) << 8);
  const float ir = inverse_scale_of(er);
  const uint64_t im = twice(inverse_scale_of(em)), back = twice(scale_of(er) * f.inv_root);
  const uint64_t decay = twice(f.decay), rate = twice(-f.rate);
  if constexpr (RANDOM_M) {
    uint32_t h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = dither_m(dither(pair + k, f.step));
    out.m.x = random_codes(f2_mul(m[0], im), f2_mul(m[1], im), h[0], h[1]);
    out.m.y = random_codes(f2_mul(m[2], im), f2_mul(m[3], im), h[2], h[3]);
  }
  float x[kLane];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // (2^-100 keeps the quotient of two zeros finite; roots of 2^-9 and more do not see it)
    float lo, hi;
    f2_unpack(f2_fma(f2_mul(v[k], twice(ir)), twice(ir), twice(0x1p-100f)), lo, hi);
    x[2 * k] = sqrt_sfu(lo);
    x[2 * k + 1] = sqrt_sfu(hi);
    f2_unpack(f2_fma(f2_pack(x[2 * k], x[2 * k + 1]), back, pair_of(c.eps)), lo, hi);
    const uint64_t quotient = f2_mul(m[k], f2_pack(rcp_approx(lo), rcp_approx(hi)));
    f2_unpack(f2_fma(quotient, rate, f2_mul(in.p.pair(k), decay)), out.p[2 * k], out.p[2 * k + 1]);
    if constexpr (!RANDOM_M) f2_unpack(f2_mul(m[k], im), mf[2 * k], mf[2 * k + 1]);
  }
  if constexpr (!RANDOM_M) out.m = pack_codes(mf);
  uint32_t h[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = dither(pair + k, f.step);
  float code[kLane];
  const float least = min3(min3(x[0], x[1], x[2]), min3(x[3], x[4], x[5]), fminf(x[6], x[7]));
  if (!round_roots(x, h, code) || !(least >= kLift)) {
#pragma unroll
    for (int e = 0; e < kLane; ++e) code[e] = round_root(vf[e], ir, e % 2 ? h[e / 2] >> 16 : h[e / 2] & 0xffffu);
  }
  out.r = pack_codes(code);
}

template <int PT, int GT, bool MASTER, bool RANDOM_M, int CAP>
__global__ void __launch_bounds__(kThreads, 3)
adamw8_kernel(const __grid_constant__ Table<CAP> tab, const __grid_constant__ RatePairs c, const int span,
              const Factors* __restrict__ factors) {
  pdl_enter();
  constexpr int WT = MASTER ? KRSI_F32 : PT;   // what the weight is read from
  const Factors f = *factors;
  if (f.skip) return;
  const int lane = threadIdx.x % 32;
  // Each warp takes `span` consecutive groups, and of them each tensor's part by itself.
  const int64_t first = (int64_t)(blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * span;
  if (first >= tab.n_chunks) return;
  int group = (int)first;
  int i = tensor_of(tab, group);
  const int end = tab.n_chunks - group < span ? tab.n_chunks : group + span;
  while (group < end) {
    while (i + 1 < tab.count && tab.t[i + 1].first_chunk <= group) ++i;
    const Tensor& t = tab.t[i];
    const int64_t at0 = (int64_t)(group - t.first_chunk) * kGroup;
    int part = min(end - group, (int)((t.n - at0 + kGroup - 1) / kGroup));
    group += part;
    const bool ragged = at0 + (int64_t)part * kGroup > t.n;   // its last group is not a whole one
    const int whole = t.aligned ? part - ragged : 0;
    using W = typename Elem<WT>::T;
    using G = typename Elem<GT>::T;
    int64_t at = at0 + lane * kLane;
    if (whole > 0) {   // with the next group's loads in flight while one is worked on
      const W* w = static_cast<const W*>(MASTER ? (const void*)t.master : t.p) + at;
      const G* g = static_cast<const G*>(t.g) + at;
      const uint8_t* m = static_cast<const uint8_t*>(t.m) + at;
      const uint8_t* r = static_cast<const uint8_t*>(t.v) + at;
      const uint8_t* ex = t.exponents + at0 / kGroup * 2;
      Lane8<WT, GT> in;
      auto fetch = [&](int j) {
        load_raw<WT>(in.p, w, (int64_t)j * kGroup, true, kLane);
        load_raw<GT>(in.g, g, (int64_t)j * kGroup, true, kLane);
        in.m = load_codes(m, (int64_t)j * kGroup, true, kLane);
        in.r = load_codes(r, (int64_t)j * kGroup, true, kLane);
        in.ex = *reinterpret_cast<const uint16_t*>(ex + 2 * j);
      };
      fetch(0);
#pragma unroll 1
      for (int j = 0; j < whole; ++j) {
        const Lane8<WT, GT> now = in;
        if (j + 1 < whole) fetch(j + 1);
        Done8 out;
        update8<WT, GT, RANDOM_M>(now, c, f, (uint32_t)((at + (int64_t)j * kGroup) >> 1), out);
        if constexpr (MASTER) store8<KRSI_F32>(const_cast<W*>(w), (int64_t)j * kGroup, true, kLane, out.p);
        store8<PT>(t.p, at + (int64_t)j * kGroup, true, kLane, out.p);
        store_codes(const_cast<uint8_t*>(m), (int64_t)j * kGroup, true, kLane, out.m);
        store_codes(const_cast<uint8_t*>(r), (int64_t)j * kGroup, true, kLane, out.r);
        if (lane == 0) *reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(ex) + 2 * j) = (uint16_t)out.ex;
      }
    }
#pragma unroll 1
    for (int j = whole; j < part; ++j) {
      const int64_t a = at + (int64_t)j * kGroup, left = t.n - a;
      const bool vec = t.aligned && left >= kLane;
      const int live = left > kLane ? kLane : (int)(left < 0 ? 0 : left);
      uint8_t* ex = t.exponents + (at0 / kGroup + j) * 2;
      Lane8<WT, GT> in;
      load_raw<WT>(in.p, MASTER ? (const void*)t.master : t.p, a, vec, live);
      load_raw<GT>(in.g, t.g, a, vec, live);
      in.m = load_codes(t.m, a, vec, live);
      in.r = load_codes(t.v, a, vec, live);
      in.ex = *reinterpret_cast<const uint16_t*>(ex);
      Done8 out;
      update8<WT, GT, RANDOM_M>(in, c, f, (uint32_t)(a >> 1), out);
      if constexpr (MASTER) store8<KRSI_F32>(t.master, a, vec, live, out.p);
      store8<PT>(t.p, a, vec, live, out.p);
      store_codes(t.m, a, vec, live, out.m);
      store_codes(t.v, a, vec, live, out.r);
      if (lane == 0) *reinterpret_cast<uint16_t*>(ex) = (uint16_t)out.ex;
    }
  }
}

// ---------------------------------------------------------------- host side
bool dtype_ok(int d) { return d == KRSI_F32 || d == KRSI_BF16 || d == KRSI_F16; }
bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int64_t launches_at_most(int64_t count) { return count / kLargeCap + 4; }   // one more for each gradient type

// A tensor's kind: what the update's kernel is compiled for.
enum States : int { kStates32 = 0, kStates8 = 1, kStates8Random = 2 };
constexpr int kKinds = 3 * 2 * 2 * 3;
constexpr int kind_of(int p_dtype, int g_dtype, bool master, int states) {
  return ((p_dtype * 2 + (g_dtype != p_dtype)) * 2 + master) * 3 + states;
}
constexpr int kBits8Random = 8 + KRSI_ADAMW_RANDOM_M;
bool in_8_bits(const krsi_adamw_tensor& t) { return t.state_bits == 8 || t.state_bits == kBits8Random; }
int kind_of(const krsi_adamw_tensor& t) {
  const int states = t.state_bits == 8 ? kStates8 : t.state_bits == kBits8Random ? kStates8Random : kStates32;
  return kind_of(t.p_dtype, t.g_dtype, t.master != nullptr, states);
}

// Calls `launch(table)` for tables of the tensors that `take` accepts, `left` of them, in chunks of `chunk` values.
template <typename Take, typename Launch>
int for_tables(const krsi_adamw_tensor* tensors, int64_t left, int chunk, Take take, Launch launch) {
  int64_t i = 0;
  auto fill = [&](auto& tab) -> int {
    constexpr int cap = sizeof(tab.t) / sizeof(tab.t[0]);
    int64_t chunks = 0;
    tab.count = 0;
    for (; left > 0 && tab.count < cap; ++i) {
      const krsi_adamw_tensor& s = tensors[i];
      if (!take(s)) continue;
      const int64_t own = (s.n + chunk - 1) / chunk;
      if (own > INT32_MAX) return KRSI_ERR_UNSUPPORTED;
      if (chunks + own > INT32_MAX) break;   // the next launch takes it
      const size_t state = in_8_bits(s) ? 8 : 32;
      const bool aligned = aligned_to(s.p, s.p_dtype == KRSI_F32 ? 32 : 16) &&
                           aligned_to(s.g, s.g_dtype == KRSI_F32 ? 32 : 16) && aligned_to(s.m, state) &&
                           aligned_to(s.v, state) && aligned_to(s.master, 32);
      tab.t[tab.count++] = Tensor{s.p, s.g, s.m, s.v, s.master, s.exponents, s.n, (int)chunks, aligned};
      chunks += own;
      --left;
    }
    tab.n_chunks = (int)chunks;
    return launch(tab);
  };
  while (left > 0) {
    int rc;
    if (left <= kSmallCap) {
      Table<kSmallCap> tab;
      rc = fill(tab);
    } else {
      Table<kLargeCap> tab;
      rc = fill(tab);
    }
    if (rc != KRSI_OK) return rc;
  }
  return KRSI_OK;
}

// How many tensors there are of each kind, and with each gradient type, and the values of each kind; tensors without
// values count for none.
struct Counts {
  int64_t kind[kKinds] = {}, grad[3] = {}, values[kKinds] = {};
};

template <int PT, int GT, bool MASTER, int STATES>
int update(const krsi_adamw_tensor* tensors, const Counts& counts, const Rates& c, const Factors* f, cudaStream_t s) {
  constexpr int kind = kind_of(PT, GT, MASTER, STATES);
  constexpr bool Q8 = STATES != kStates32;
  auto take = [](const krsi_adamw_tensor& t) { return t.n > 0 && kind_of(t) == kind; };
  // fp32 states: one group a warp where four would leave SMs without a block (150,000 values: 5 us became 3)
  const int groups = counts.values[kind] < (int64_t)kNumSMsB200 * kChunk ? 1 : kGroupsPerWarp;
  const int chunk = Q8 ? kGroup : kThreads / 32 * groups * kGroup;
  return for_tables(tensors, counts.kind[kind], chunk, take, [&](const auto& tab) -> int {
    constexpr int cap = sizeof(tab.t) / sizeof(tab.t[0]);
    if constexpr (Q8) {
      // consecutive groups in equal shares (16 at a time, in turns, take 10% more)
      constexpr int warps = kBlocks8 * (kThreads / 32);
      const int64_t span = ((int64_t)tab.n_chunks + warps - 1) / warps;
      const int64_t blocks = (tab.n_chunks + span * (kThreads / 32) - 1) / (span * (kThreads / 32));
      KRSI_CUDA_TRY(launch_pdl(adamw8_kernel<PT, GT, MASTER, STATES == kStates8Random, cap>, dim3((unsigned)blocks),
                               dim3(kThreads), 0, s, tab, RatePairs(c), (int)span, f));
    } else {
      KRSI_CUDA_TRY(launch_pdl(adamw_kernel<PT, GT, MASTER, cap>, dim3(tab.n_chunks), dim3(kThreads), 0, s, tab, c, groups,
                               f));
    }
    return KRSI_OK;
  });
}

template <int GT>
int norm(const krsi_adamw_tensor* tensors, const Counts& counts, double* partial, int64_t room, int* used,
         cudaStream_t s) {
  auto take = [](const krsi_adamw_tensor& t) { return t.n > 0 && t.g_dtype == GT; };
  return for_tables(tensors, counts.grad[GT], kChunk, take, [&](const auto& tab) -> int {
    constexpr int cap = sizeof(tab.t) / sizeof(tab.t[0]);
    const int blocks = tab.n_chunks < kNormBlocks ? tab.n_chunks : kNormBlocks;
    if (*used + blocks > room) return KRSI_ERR_WORKSPACE;
    KRSI_CUDA_TRY(launch_pdl(adamw_norm_kernel<GT, cap>, dim3(blocks), dim3(kThreads), 0, s, tab, partial + *used));
    *used += blocks;
    return KRSI_OK;
  });
}

}  // namespace
}  // namespace krsi

using namespace krsi;

extern "C" int krsi_adamw_workspace_size(int64_t count, size_t* bytes) {
  KRSI_CHECK_ARG(count >= 0 && bytes);
  *bytes = kFactorBytes + (size_t)(launches_at_most(count) * kNormBlocks) * sizeof(double);
  return KRSI_OK;
}

extern "C" int krsi_adamw_step(const krsi_adamw_tensor* tensors, int64_t count, int64_t* step, const float* lr_dev,
                               double lr, double beta1, double beta2, double eps, double weight_decay, double max_norm,
                               float* norm_out, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  KRSI_CHECK_ARG(count >= 0 && (count == 0 || tensors) && step);
  KRSI_CHECK_ARG(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && max_norm >= 0);
  KRSI_CHECK_ARG(max_norm == 0 || ((float)max_norm > 0 && norm_out));
  Counts counts;
  for (int64_t i = 0; i < count; ++i) {
    const krsi_adamw_tensor& t = tensors[i];
    KRSI_CHECK_ARG(t.n >= 0 && dtype_ok(t.p_dtype) && (t.state_bits == 32 || in_8_bits(t)));
    KRSI_CHECK_ARG(t.g_dtype == t.p_dtype || t.g_dtype == KRSI_F32);
    if (t.n == 0) continue;
    KRSI_CHECK_ARG(t.p && t.g && t.m && t.v && (t.state_bits == 32 || t.exponents));
    KRSI_CHECK_ARG(t.p_dtype != KRSI_F32 || !t.master);
    if (in_8_bits(t) && !aligned_to(t.exponents, 2)) return KRSI_ERR_MISALIGNED;
    ++counts.kind[kind_of(t)];
    ++counts.grad[t.g_dtype];
    counts.values[kind_of(t)] += t.n;
  }
  size_t need = 0;
  krsi_adamw_workspace_size(count, &need);
  if (!workspace || workspace_bytes < need) return KRSI_ERR_WORKSPACE;
  if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  Factors* factors = static_cast<Factors*>(workspace);
  double* partial = reinterpret_cast<double*>(static_cast<char*>(workspace) + kFactorBytes);
  int used = 0;
  if (max_norm > 0) {
    const int64_t room = launches_at_most(count) * kNormBlocks;
    int rc = norm<KRSI_F32>(tensors, counts, partial, room, &used, stream);
    if (rc == KRSI_OK) rc = norm<KRSI_BF16>(tensors, counts, partial, room, &used, stream);
    if (rc == KRSI_OK) rc = norm<KRSI_F16>(tensors, counts, partial, room, &used, stream);
    if (rc != KRSI_OK) return rc;
  }
  const FactorArgs fa{partial, used, norm_out, step, lr_dev, lr, log(beta1), log(beta2), weight_decay, (float)max_norm};
  KRSI_CUDA_TRY(launch_pdl(adamw_factors_kernel, dim3(1), dim3(256), 0, stream, fa, factors));
  const Rates c{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
#define KRSI_UPDATE(PT, GT, MASTER)                                                        \
  do {                                                                                     \
    int rc = update<PT, GT, MASTER, kStates32>(tensors, counts, c, factors, stream);       \
    if (rc == KRSI_OK) rc = update<PT, GT, MASTER, kStates8>(tensors, counts, c, factors, stream); \
    if (rc == KRSI_OK) rc = update<PT, GT, MASTER, kStates8Random>(tensors, counts, c, factors, stream); \
    if (rc != KRSI_OK) return rc;                                                          \
  } while (0)
  KRSI_UPDATE(KRSI_F32, KRSI_F32, false);
  KRSI_UPDATE(KRSI_BF16, KRSI_BF16, false);
  KRSI_UPDATE(KRSI_BF16, KRSI_BF16, true);
  KRSI_UPDATE(KRSI_BF16, KRSI_F32, false);
  KRSI_UPDATE(KRSI_BF16, KRSI_F32, true);
  KRSI_UPDATE(KRSI_F16, KRSI_F16, false);
  KRSI_UPDATE(KRSI_F16, KRSI_F16, true);
  KRSI_UPDATE(KRSI_F16, KRSI_F32, false);
  KRSI_UPDATE(KRSI_F16, KRSI_F32, true);
#undef KRSI_UPDATE
  return KRSI_OK;
}
