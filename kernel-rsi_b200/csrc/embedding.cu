// embedding.cu - the embedding lookup with scaling, and the table's gradient by sorted tokens.
//   forward:  out[i] = scale * table[tokens[i]]                       (a gather)
//   backward: dtable[v] = scale * sum over i with tokens[i] = v of g[i], in a fixed order (that of token_rows.cu's
//             sort; the positions' own up to 512 of them)
// Both are bound by memory: the forward reads the looked-up rows and writes out; the backward reads g
// once and writes every row of dtable once (zeros for tokens that do not occur).
//
// Measured at 32768 rows of 1152 bf16 values, vocabulary 32768 (B200): lookup 22 us (15 us at the copy rate), gradient
// 50 us (24): the sort 12 us, which waits on L2, the sums 33, the long runs 6.  The lookup's rows are staged by
// asynchronous copies; held in registers it took 34 us, too little being in flight.
//
// A token id outside [0, V) reads nothing: its row of out is NaN and it adds to no gradient.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "token_rows.cuh"

namespace krsi {
namespace {

using tokens::Pack;

template <int DT>
__device__ __forceinline__ typename Elem<DT>::T nan_of() { return Elem<DT>::store(__int_as_float(0x7fffffff)); }

// ---------------------------------------------------------------- forward
// A thread keeps one packet of columns and takes up to kFwdRows rows, staged in shared memory so that
// their loads are in flight together (behind those of their tokens).
constexpr int kFwdRows = 16;

template <int DT, int VEC, typename I>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const I* __restrict__ toks, const typename Elem<DT>::T* __restrict__ table,
                     typename Elem<DT>::T* __restrict__ out, int n, int rows, uint32_t packets, int64_t V, float scale) {
  pdl_enter();
  using E = Elem<DT>;
  using P = Pack<typename E::T, VEC>;
  const uint32_t c = blockIdx.y * blockDim.x + threadIdx.x;
  const int row0 = (int)blockIdx.x * rows, m = min(rows, n - row0);
  __shared__ int s_tok[kFwdRows];    // -1: outside the table
  if (threadIdx.x < m) {
    const I v = toks[row0 + threadIdx.x];
    s_tok[threadIdx.x] = v >= 0 && v < (I)V ? (int)v : -1;
  }
  __syncthreads();
  if (c >= packets) return;
  extern __shared__ __align__(16) unsigned char stage_raw[];
  P* stage = reinterpret_cast<P*>(stage_raw) + threadIdx.x;   // [rows][blockDim.x]
  const P* tp = reinterpret_cast<const P*>(table) + c;
  P* op = reinterpret_cast<P*>(out) + (int64_t)row0 * packets + c;
  P none;
#pragma unroll
  for (int e = 0; e < VEC; ++e) none.v[e] = nan_of<DT>();
#pragma unroll 4
  for (int k = 0; k < m; ++k) {
    const int t = s_tok[k];
    if (t >= 0) tokens::copy_packet(stage + k * blockDim.x, tp + (int64_t)t * packets);
    else stage[k * blockDim.x] = none;
  }
  tokens::copy_commit();
  tokens::copy_wait<0>();
#pragma unroll 4
  for (int k = 0; k < m; ++k) {
    P r = stage[k * blockDim.x];
    if (scale != 1.0f) {   // else the row's own bits
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = E::store(scale * E::load(r.v[e]));
    }
    op[(int64_t)k * packets] = r;
  }
}

// ---------------------------------------------------------------- backward
// Where the sums by token go: dtable rows, scaled and rounded once (zeros for tokens that do not occur).
template <int DT, int VEC>
struct TableRows {
  using T = typename Elem<DT>::T;
  T* dtable;
  int64_t d;
  float scale;
  static constexpr bool kUsesFirst = false;
  using Base = tokens::NoBase;
  __device__ __forceinline__ Base fetch(int, int, uint32_t) const { return {}; }
  __device__ __forceinline__ void packet(int v, uint32_t c, const float* sums, Base) const {
    Pack<T, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = Elem<DT>::store(scale * sums[e]);
    *reinterpret_cast<Pack<T, VEC>*>(dtable + v * d + c * VEC) = o;
  }
  __device__ __forceinline__ void zero(int v, uint32_t c) const {
    Pack<T, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = Elem<DT>::store(0.f);
    *reinterpret_cast<Pack<T, VEC>*>(dtable + v * d + c * VEC) = o;
  }
  __device__ __forceinline__ void column(int v, int, int col, float sum) const {
    dtable[v * d + col] = Elem<DT>::store(scale * sum);
  }
};

// Elements per packet: the widest access that divides the row and suits both buffers' alignment.
template <typename T>
int packet_elems(int64_t d, const void* a, const void* b) {
  int vec = 16 / (int)sizeof(T);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b);
  while (vec > 1 && (d % vec != 0 || bits % (vec * sizeof(T)) != 0)) vec /= 2;
  return vec;
}

template <int DT, int VEC>
int fwd(const void* toks, int token_bits, const void* table, void* out, int64_t n, int64_t V, int64_t d, float scale,
        cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const uint32_t packets = (uint32_t)(d / VEC);
  const int threads = (int)std::min<uint32_t>(256, std::max<uint32_t>(32, (packets + 31) / 32 * 32));
  // as many rows a block as still leave a block for every SM
  const int rows = (int)std::max<int64_t>(1, std::min<int64_t>(kFwdRows, n / kNumSMsB200));
  const dim3 grid((unsigned)((n + rows - 1) / rows), (packets + threads - 1) / threads);
  const size_t smem = (size_t)rows * threads * VEC * sizeof(T);   // at most 64 KB
  auto launch = [&](auto* t) -> int {
    using I = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    constexpr auto kern = embedding_fwd_kernel<DT, VEC, I>;
    KRSI_CUDA_TRY(allow_smem<kern>(kFwdRows * 256 * 16));
    KRSI_CUDA_TRY(launch_pdl(kern, grid, dim3(threads), smem, stream, t, (const T*)table, (T*)out, (int)n, rows,
                             packets, V, scale));
    return KRSI_OK;
  };
  return token_bits == 64 ? launch((const long long*)toks) : launch((const int*)toks);
}

template <int DT, int VEC>
int bwd(const void* toks, int token_bits, const void* g, const tokens::Space& s, void* dtable, int64_t n, int64_t V,
        int64_t d, float scale, int64_t padding_idx, cudaStream_t stream) {
  const TableRows<DT, VEC> rows{(typename Elem<DT>::T*)dtable, d, scale};
  if (n <= tokens::kFewRows) {
    KRSI_CUDA_TRY(token_bits == 64
                      ? (tokens::sum_few<DT, VEC, false>(g, nullptr, (const long long*)toks, rows, true, n, V,
                                                         padding_idx, d, stream))
                      : (tokens::sum_few<DT, VEC, false>(g, nullptr, (const int*)toks, rows, true, n, V, padding_idx, d,
                                                         stream)));
    return KRSI_OK;
  }
  KRSI_CUDA_TRY(tokens::token_sort(toks, token_bits, n, V, padding_idx, s.start, s.pos, s.tok, stream));
  KRSI_CUDA_TRY((tokens::sum_by_token<DT, VEC, false>(g, nullptr, s, rows, true, n, V, d, stream)));
  return KRSI_OK;
}

// Runs fn<DT, VEC>(...) for a dtype code and a packet width.
#define KRSI_EMB_VEC(FN, DT, vec, ...)           \
  switch (vec) {                                 \
    case 8: if constexpr (DT != KRSI_F32) return FN<DT, 8>(__VA_ARGS__); [[fallthrough]]; \
    case 4: return FN<DT, 4>(__VA_ARGS__);       \
    case 2: return FN<DT, 2>(__VA_ARGS__);       \
    default: return FN<DT, 1>(__VA_ARGS__);      \
  }
#define KRSI_EMB_DISPATCH(FN, a, b, ...)                                                                   \
  switch (dtype) {                                                                                         \
    case KRSI_F32: KRSI_EMB_VEC(FN, KRSI_F32, packet_elems<float>(d, a, b), __VA_ARGS__)                   \
    case KRSI_BF16: KRSI_EMB_VEC(FN, KRSI_BF16, packet_elems<__nv_bfloat16>(d, a, b), __VA_ARGS__)         \
    default: KRSI_EMB_VEC(FN, KRSI_F16, packet_elems<__half>(d, a, b), __VA_ARGS__)                        \
  }

inline int check(int64_t n, int64_t V, int64_t d, int token_bits, int dtype) {
  KRSI_CHECK_ARG(n >= 0 && V > 0 && d > 0);
  KRSI_CHECK_ARG(token_bits == 32 || token_bits == 64);
  KRSI_CHECK_ARG(dtype == KRSI_F32 || dtype == KRSI_BF16 || dtype == KRSI_F16);
  // 32-bit positions and tokens in the sort; a grid dimension of column blocks
  if (n > INT32_MAX / 2 || V > INT32_MAX - 1024 || d > 65535 * 32) return KRSI_ERR_UNSUPPORTED;
  return KRSI_OK;
}

}  // namespace
}  // namespace krsi

using namespace krsi;

extern "C" int krsi_embedding_fwd(const void* toks, int token_bits, const void* table, void* out, int64_t n,
                                  int64_t V, int64_t d, float scale, int dtype, cudaStream_t stream) {
  const int rc = check(n, V, d, token_bits, dtype);
  if (rc != KRSI_OK) return rc;
  if (n == 0) return KRSI_OK;
  KRSI_CHECK_ARG(toks && table && out);
  KRSI_EMB_DISPATCH(fwd, table, out, toks, token_bits, table, out, n, V, d, scale, stream)
}

extern "C" int krsi_embedding_bwd_workspace_size(int64_t n, int64_t V, int64_t d, size_t* bytes) {
  KRSI_CHECK_ARG(bytes && n >= 0 && V > 0 && d > 0);
  *bytes = tokens::space_at(nullptr, n, V, d).bytes;
  return KRSI_OK;
}

extern "C" int krsi_embedding_bwd(const void* toks, int token_bits, const void* g, void* dtable, void* workspace,
                                  size_t workspace_bytes, int64_t n, int64_t V, int64_t d, float scale,
                                  int64_t padding_idx, int dtype, cudaStream_t stream) {
  const int rc = check(n, V, d, token_bits, dtype);
  if (rc != KRSI_OK) return rc;
  KRSI_CHECK_ARG(dtable && padding_idx < V);
  if (n == 0) {   // no row was looked up: the table's gradient is zero
    KRSI_CUDA_TRY(cudaMemsetAsync(dtable, 0, (size_t)V * d * (dtype == KRSI_F32 ? 4 : 2), stream));
    return KRSI_OK;
  }
  KRSI_CHECK_ARG(toks && g);
  const tokens::Space s = tokens::space_at(workspace, n, V, d);
  if (!workspace || workspace_bytes < s.bytes) return KRSI_ERR_WORKSPACE;
  if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  KRSI_EMB_DISPATCH(bwd, g, dtable, toks, token_bits, g, s, dtable, n, V, d, scale, padding_idx, stream)
}
