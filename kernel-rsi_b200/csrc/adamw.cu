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
// v, because a square takes twice the binades.  m is rounded to nearest: it moves by a tenth a step, more than half
// a code.  v moves by a thousandth, far less than half a code: rounded to nearest it would stay where it is, so r
// is rounded up or down at random, right on average.  The randomness is a hash of the element's place and t, so a
// step has the same bits every time.  A positive v never becomes 0, which eps alone would divide by.
// A group with a value that is not finite reads back as NaN.
// The moments and their codes are formed by IEEE operations in a fixed order without contraction.
#include <math.h>

#include <cuda_fp8.h>

#include "common.cuh"

namespace krsi {
namespace {

constexpr int kGroup = 256;                        // values that share the exponents of 8-bit states
constexpr int kThreads = 256;
constexpr int kGroupsPerWarp = 4;
constexpr int kChunk = kThreads / 32 * kGroupsPerWarp * kGroup;   // values of one block: 8192
constexpr int kLane = 8;                           // values of one lane
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
  int first_chunk;   // chunks of the tensors before it in the launch
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

// ---------------------------------------------------------------- eight codes
__device__ __forceinline__ void decode8(const void* base, int64_t at, bool vec, int live, float scale, float* o) {
  const uint8_t* p = static_cast<const uint8_t*>(base) + at;
  uint32_t u[2] = {0, 0};
  if (vec) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    u[0] = w.x;
    u[1] = w.y;
  } else {
#pragma unroll
    for (int e = 0; e < kLane; ++e)
      if (e < live) u[e / 4] |= (uint32_t)p[e] << (8 * (e % 4));
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __half2_raw h =
        __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((u[k / 2] >> (16 * (k % 2))) & 0xffff), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    o[2 * k] = __fmul_rn(f.x, scale);
    o[2 * k + 1] = __fmul_rn(f.y, scale);
  }
}
__device__ __forceinline__ void encode8(void* base, int64_t at, bool vec, int live, const float* o) {
  uint8_t* p = static_cast<uint8_t*>(base) + at;
  uint32_t u[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    u[k / 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(o[2 * k], o[2 * k + 1]), __NV_SATFINITE, __NV_E4M3)
                << (16 * (k % 2));
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
  } else {
#pragma unroll
    for (int e = 0; e < kLane; ++e)
      if (e < live) p[e] = (uint8_t)(u[e / 4] >> (8 * (e % 4)));
  }
}
// 2^(byte - 127), NaN for the mark of a group that is not finite.
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fffffffu : byte << 23);
}
// 2^(127 - byte)
__device__ __forceinline__ float inverse_scale_of(uint32_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fffffffu : (254 - byte) << 23);
}
// 16 random bits for each of a pair of places (low half: the even one).
__device__ __forceinline__ uint32_t dither(uint32_t pair, uint32_t step) {
  uint32_t h = pair * 0x9E3779B1u + step * 0x632BE5ABu;
  h = (h ^ (h >> 16)) * 0x21F0AAADu;
  h = (h ^ (h >> 15)) * 0x735A2D97u;
  return h ^ (h >> 15);
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
  if (threadIdx.x != 0) return;
  Factors f{1.f, 0.f, 0.f, 0.f, 0u, 0};
  if (a.max_norm > 0.f) {
    double total = 0.0;
    for (int i = 0; i < 8; ++i) total += red[i];
    const float norm = (float)sqrt(total);
    if (a.norm) *a.norm = norm;
    f.clip = fminf(__fdiv_rn(a.max_norm, __fadd_rn(norm, 1e-6f)), 1.f);
    f.skip = !isfinite(norm);
  }
  if (!f.skip) {
    const int64_t t = *a.step + 1;
    *a.step = t;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    f.rate = (float)(lr / -expm1((double)t * a.log_beta1));
    f.inv_root = (float)(1.0 / sqrt(-expm1((double)t * a.log_beta2)));
    f.decay = (float)(1.0 - lr * a.decay);
    f.step = (uint32_t)t;
  }
  *out = f;
}

struct Rates {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps;
};

template <int PT, int GT, bool MASTER, bool Q8, int CAP>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(const __grid_constant__ Table<CAP> tab, const Rates c, const Factors* __restrict__ factors) {
  pdl_enter();
  const Factors f = *factors;
  if (f.skip) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Tensor& t = tab.t[tensor_of(tab, blockIdx.x)];
  const int64_t base = (int64_t)(blockIdx.x - t.first_chunk) * kChunk + warp * (kGroupsPerWarp * kGroup);
  const int64_t n = t.n;
#pragma unroll 1
  for (int j = 0; j < kGroupsPerWarp; ++j) {
    const int64_t at0 = base + j * kGroup;   // the group's first value
    if (at0 >= n) return;
    const int64_t at = at0 + lane * kLane, left = n - at;
    const bool vec = t.aligned && left >= kLane;
    const int live = left > kLane ? kLane : (int)(left < 0 ? 0 : left);
    float p[kLane], g[kLane], m[kLane], v[kLane];
    if constexpr (MASTER) load8<KRSI_F32>(t.master, at, vec, live, p);
    else load8<PT>(t.p, at, vec, live, p);
    load8<GT>(t.g, at, vec, live, g);
    if constexpr (Q8) {
      const uint8_t* ex = t.exponents + at0 / kGroup * 2;
      const float sm = scale_of(ex[0]), sr = scale_of(ex[1]);
      decode8(t.m, at, vec, live, sm, m);
      decode8(t.v, at, vec, live, sr, v);
#pragma unroll
      for (int e = 0; e < kLane; ++e) v[e] = __fmul_rn(v[e], v[e]);
    } else {
      load8<KRSI_F32>(t.m, at, vec, live, m);
      load8<KRSI_F32>(t.v, at, vec, live, v);
    }
    float r[kLane];
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      const float ge = __fmul_rn(g[e], f.clip);
      m[e] = __fadd_rn(__fmul_rn(m[e], c.beta1), __fmul_rn(ge, c.one_minus_beta1));
      v[e] = __fadd_rn(__fmul_rn(v[e], c.beta2), __fmul_rn(__fmul_rn(ge, ge), c.one_minus_beta2));
      r[e] = __fsqrt_rn(v[e]);
      p[e] = p[e] * f.decay - f.rate * __fdividef(m[e], fmaf(r[e], f.inv_root, c.eps));
    }
    if constexpr (MASTER) store8<KRSI_F32>(t.master, at, vec, live, p);
    store8<PT>(t.p, at, vec, live, p);
    if constexpr (Q8) {
      uint32_t top_m = 0, top_v = 0;
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        top_m = max(top_m, __float_as_uint(m[e]) & 0x7fffffffu);
        top_v = max(top_v, __float_as_uint(v[e]) & 0x7fffffffu);
      }
      const int field_m = (int)(__reduce_max_sync(0xffffffffu, top_m) >> 23);
      const int field_v = (int)(__reduce_max_sync(0xffffffffu, top_v) >> 23);
      // the group's largest magnitude 2^k f, 1 <= f < 2, becomes 2^7 f
      const uint32_t em = field_m == 255 ? 255u : (uint32_t)max(field_m - 7, 1);
      const uint32_t er = field_v == 255 ? 255u : (uint32_t)(((field_v - 127) >> 1) + 120);
      const float im = inverse_scale_of(em), ir = inverse_scale_of(er);
#pragma unroll
      for (int e = 0; e < kLane; e += 2) {
        const uint32_t h = dither((uint32_t)(at >> 1) + e / 2, f.step);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          m[e + k] = __fmul_rn(m[e + k], im);
          // up with the probability of the bits below the code's last one: they and the random bits carry into it.
          // (Below 2^-6 codes are 2^-9 apart: 2^-6 more puts the sum where fp32's 20th bit is worth that.)
          const float x = __fmul_rn(r[e + k], ir);
          const float lift = x < 0.015625f ? 0.015625f : 0.f;
          const uint32_t random = k == 0 ? (h & 0xffffu) << 4 : (h >> 16) << 4;
          const uint32_t up = (__float_as_uint(__fadd_rn(x, lift)) + random) & 0xfff00000u;
          r[e + k] = x > 0.f ? fmaxf(__fadd_rn(__uint_as_float(up), -lift), 0.001953125f) : 0.f;
        }
      }
      encode8(t.m, at, vec, live, m);
      encode8(t.v, at, vec, live, r);
      if (lane == 0) *reinterpret_cast<uint16_t*>(t.exponents + at0 / kGroup * 2) = (uint16_t)(em | (er << 8));
    } else {
      store8<KRSI_F32>(t.m, at, vec, live, m);
      store8<KRSI_F32>(t.v, at, vec, live, v);
    }
  }
}

// ---------------------------------------------------------------- host side
bool dtype_ok(int d) { return d == KRSI_F32 || d == KRSI_BF16 || d == KRSI_F16; }
bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int64_t launches_at_most(int64_t count) { return count / kLargeCap + 4; }   // one more for each gradient type

// Calls `launch(table, first, n)` for tables of the tensors that `take` accepts, as few as their number allows.
template <typename Take, typename Launch>
int for_tables(const krsi_adamw_tensor* tensors, int64_t count, Take take, Launch launch) {
  int64_t i = 0;
  while (i < count) {
    int n = 0;
    for (int64_t j = i; j < count && n <= kSmallCap; ++j) n += take(tensors[j]) && tensors[j].n > 0;
    if (n == 0) return KRSI_OK;
    auto fill = [&](auto& tab) -> int {
      constexpr int cap = sizeof(tab.t) / sizeof(tab.t[0]);
      int64_t chunks = 0;
      tab.count = 0;
      for (; i < count && tab.count < cap; ++i) {
        const krsi_adamw_tensor& s = tensors[i];
        if (!take(s) || s.n == 0) continue;
        const int64_t own = (s.n + kChunk - 1) / kChunk;
        if (own > INT32_MAX) return KRSI_ERR_UNSUPPORTED;
        if (chunks + own > INT32_MAX) break;   // the next launch takes it
        Tensor& t = tab.t[tab.count++];
        t = Tensor{s.p, s.g, s.m, s.v, s.master, s.exponents, s.n, (int)chunks, 0};
        const size_t state = s.state_bits == 8 ? 8 : 32;
        t.aligned = aligned_to(s.p, s.p_dtype == KRSI_F32 ? 32 : 16) && aligned_to(s.g, s.g_dtype == KRSI_F32 ? 32 : 16) &&
                    aligned_to(s.m, state) && aligned_to(s.v, state) && aligned_to(s.master, 32);
        chunks += own;
      }
      tab.n_chunks = (int)chunks;
      return launch(tab);
    };
    int rc;
    if (n <= kSmallCap) {
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

template <int PT, int GT, bool MASTER, bool Q8>
int update(const krsi_adamw_tensor* tensors, int64_t count, const Rates& c, const Factors* f, cudaStream_t s) {
  return for_tables(
      tensors, count,
      [](const krsi_adamw_tensor& t) {
        return t.p_dtype == PT && t.g_dtype == GT && (t.master != nullptr) == MASTER && (t.state_bits == 8) == Q8;
      },
      [&](const auto& tab) -> int {
        constexpr int cap = sizeof(tab.t) / sizeof(tab.t[0]);
        KRSI_CUDA_TRY(launch_pdl(adamw_kernel<PT, GT, MASTER, Q8, cap>, dim3(tab.n_chunks), dim3(kThreads), 0, s, tab, c, f));
        return KRSI_OK;
      });
}

template <int GT>
int norm(const krsi_adamw_tensor* tensors, int64_t count, double* partial, int64_t room, int* used, cudaStream_t s) {
  return for_tables(
      tensors, count, [](const krsi_adamw_tensor& t) { return t.g_dtype == GT; },
      [&](const auto& tab) -> int {
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
  KRSI_CHECK_ARG(max_norm == 0 || norm_out);
  for (int64_t i = 0; i < count; ++i) {
    const krsi_adamw_tensor& t = tensors[i];
    KRSI_CHECK_ARG(t.n >= 0 && dtype_ok(t.p_dtype) && (t.state_bits == 8 || t.state_bits == 32));
    KRSI_CHECK_ARG(t.g_dtype == t.p_dtype || t.g_dtype == KRSI_F32);
    if (t.n == 0) continue;
    KRSI_CHECK_ARG(t.p && t.g && t.m && t.v && (t.state_bits == 32 || t.exponents));
    KRSI_CHECK_ARG(t.p_dtype != KRSI_F32 || !t.master);
    if (t.state_bits == 8 && !aligned_to(t.exponents, 2)) return KRSI_ERR_MISALIGNED;
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
    int rc = norm<KRSI_F32>(tensors, count, partial, room, &used, stream);
    if (rc == KRSI_OK) rc = norm<KRSI_BF16>(tensors, count, partial, room, &used, stream);
    if (rc == KRSI_OK) rc = norm<KRSI_F16>(tensors, count, partial, room, &used, stream);
    if (rc != KRSI_OK) return rc;
  }
  const FactorArgs fa{partial, used, norm_out, step, lr_dev, lr, log(beta1), log(beta2), weight_decay, (float)max_norm};
  KRSI_CUDA_TRY(launch_pdl(adamw_factors_kernel, dim3(1), dim3(256), 0, stream, fa, factors));
  const Rates c{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
#define KRSI_UPDATE(PT, GT, MASTER)                                                        \
  do {                                                                                     \
    int rc = update<PT, GT, MASTER, false>(tensors, count, c, factors, stream);            \
    if (rc == KRSI_OK) rc = update<PT, GT, MASTER, true>(tensors, count, c, factors, stream); \
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
