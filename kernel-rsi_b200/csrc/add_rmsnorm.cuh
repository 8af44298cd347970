// add_rmsnorm.cuh - what the residual norm's forward and backward share: a row's packets and how rows of any width
// are spread over threads.
#pragma once
#include <initializer_list>

#include "common.cuh"

namespace krsi {
namespace norm {

// Four values of 16 bits (rows of whole 8 bytes).
template <typename T>
struct alignas(8) Vec8 {
  T v[4];
};

template <int DT, int VEC>
__device__ __forceinline__ void load_row(const typename Elem<DT>::T* p, float* out, bool stream) {
  using E = Elem<DT>;
  if constexpr (VEC == 1) {
    out[0] = E::load(*p);
  } else if constexpr (VEC * sizeof(typename E::T) == 8) {
    const auto v = *reinterpret_cast<const Vec8<typename E::T>*>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = E::load(v.v[k]);
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
  } else if constexpr (VEC * sizeof(typename E::T) == 8) {
    Vec8<typename E::T> o;
#pragma unroll
    for (int k = 0; k < 4; ++k) o.v[k] = E::store(in[k]);
    *reinterpret_cast<Vec8<typename E::T>*>(p) = o;
  } else {
    Vec16<typename E::T> o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.v[k] = E::store(in[k]);
    stg16(p, o);
  }
}
// w's values, of the rows' type or fp32.
template <int DT, int VEC>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int col, float* out) {
  if (DT == KRSI_F32 || f32) {
    const float* p = static_cast<const float*>(w) + col;
    if constexpr (VEC == 1) {
      out[0] = __ldg(p);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + e));
        out[e] = v.x; out[e + 1] = v.y; out[e + 2] = v.z; out[e + 3] = v.w;
      }
    }
  } else {
    load_row<DT, VEC>(static_cast<const typename Elem<DT>::T*>(w) + col, out, false);
  }
}

// The widest packets, in values, that rows of n values at these addresses allow: 16 or 8 bytes, or 1 value.  A packet's
// values of w are as many bytes as the row's, or in fp32 beside 16 bits 16 at a time.
inline int packet_of(int x_dtype, int w_dtype, int64_t n, const void* w, std::initializer_list<const void*> rows) {
  const int es = x_dtype == KRSI_F32 ? 4 : 2;
  for (int bytes : {16, 8}) {
    if (es == 4 && bytes == 8) break;
    auto on = [](const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; };
    bool ok = n * es % bytes == 0 && on(w, w_dtype == KRSI_F32 ? 16 : bytes);
    for (const void* p : rows) ok = ok && on(p, bytes);
    if (ok) return bytes / es;
  }
  return 1;
}

inline bool dtype_ok(int d) { return d == KRSI_F32 || d == KRSI_BF16 || d == KRSI_F16; }
// w has x's type, or is fp32.
inline bool types_ok(int x_dtype, int w_dtype) { return w_dtype == x_dtype || w_dtype == KRSI_F32; }

}  // namespace norm
}  // namespace krsi
