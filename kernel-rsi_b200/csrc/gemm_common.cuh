// gemm_common.cuh - what the hand-written tcgen05 GEMMs share: 2-D tensor maps, operand descriptors and
// the wind-down of the TMA ring.
#pragma once
#include <string.h>

#include "attn_common.cuh"
#include "sm100.cuh"

namespace krsi {
namespace gemm {

using namespace sm100;

// After an abort: wait (bounded) until the last kStages K blocks the producer issued have landed, so
// no TMA load is still writing this CTA's shared memory when it exits.
template <int S>
__device__ __forceinline__ void drain_loads(uint64_t* full, int issued, uint32_t limit) {
  for (int j = issued > S ? issued - S : 0; j < issued; ++j) {
    for (uint32_t n = 0; n < limit && !mbar_try_wait(&full[j % S], (j / S) & 1); ++n) {
    }
  }
}

// K-major operand in the 128-byte swizzle: 8-row groups of 8 x 128 B (SBO = 1024 B); the K step of
// 16 elements inside the swizzle row advances the start address by 32 B.
__device__ __forceinline__ uint64_t kmajor_sw128(uint32_t addr) { return smem_desc(addr, 16, 1024, kSw128); }

// The tensor maps are made by the driver API, which wants a context current to the calling thread; a
// thread that has made no runtime call yet (an autograd worker) may have none.  Gives it the primary one
// then (cudaSetDevice, which stream capture allows), and leaves a context that is there alone.
inline cudaError_t bind_context() {
  using GetCurrent = CUresult (*)(CUcontext*);
  static GetCurrent get = nullptr;
  if (!get) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    const cudaError_t e = cudaGetDriverEntryPoint("cuCtxGetCurrent", &p, cudaEnableDefault, &q);
    if (e != cudaSuccess) return e;
    if (q != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
    get = reinterpret_cast<GetCurrent>(p);
  }
  CUcontext ctx = nullptr;
  if (get(&ctx) == CUDA_SUCCESS && ctx != nullptr) return cudaSuccess;
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  return e != cudaSuccess ? e : cudaSetDevice(dev);
}

// 2-D view (cols, rows) of a row-major 16-bit matrix with `pitch` elements between rows, copied in
// boxes of box_cols x box_rows with the given swizzle.  Loads read elements past cols or rows as
// zero; stores skip them.
inline bool make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch, bool f16,
              uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  attn::EncodeTiledFn enc = attn::encode_fn();
  if (!enc) return false;
  memset(map, 0, sizeof(*map));
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch * 2};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                   const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}
}  // namespace gemm
}  // namespace krsi
