// embedding.cu - the embedding lookup with scaling, and the table's gradient by sorted tokens.
//   forward:  out[i] = scale * table[tokens[i]]                       (a gather)
//   backward: dtable[v] = scale * sum over i with tokens[i] = v of g[i], in position order
// Both are bound by memory: the forward reads the looked-up rows and writes out; the backward reads g
// once and writes every row of dtable once (zeros for tokens that do not occur).
//
// A token id outside [0, V) reads nothing: its row of out is NaN and it adds to no gradient.
#include <algorithm>

#include "common.cuh"
#include "token_rows.cuh"

namespace krsi {
namespace {

using tokens::kChunkRows;

// VEC elements moved as one access (16, 8, 4 or 2 bytes).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <int DT>
__device__ __forceinline__ typename Elem<DT>::T nan_of() { return Elem<DT>::store(__int_as_float(0x7fffffff)); }

// ---------------------------------------------------------------- forward
// One packet per work item, kFwdItems items per thread with their loads in flight together.
constexpr int kFwdItems = 4;

template <int DT, int VEC, typename I>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const I* __restrict__ toks, const typename Elem<DT>::T* __restrict__ table,
                     typename Elem<DT>::T* __restrict__ out, int64_t items, uint32_t packets, int64_t V, float scale) {
  pdl_enter();
  using E = Elem<DT>;
  using P = Pack<typename E::T, VEC>;
  const P* tp = reinterpret_cast<const P*>(table);
  P* op = reinterpret_cast<P*>(out);
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i0 < items; i0 += kFwdItems * stride) {
    P r[kFwdItems];
#pragma unroll
    for (int k = 0; k < kFwdItems; ++k) {
      const int64_t i = i0 + k * stride;
      if (i >= items) break;
      const int64_t row = i / packets;
      const uint32_t c = (uint32_t)(i - row * packets);
      const int64_t t = toks[row];
      if (t >= 0 && t < V) {
        r[k] = tp[t * packets + c];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[k].v[e] = nan_of<DT>();
      }
    }
#pragma unroll
    for (int k = 0; k < kFwdItems; ++k) {
      const int64_t i = i0 + k * stride;
      if (i >= items) break;
      if (scale != 1.0f) {   // else the row's own bits
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[k].v[e] = E::store(scale * E::load(r[k].v[e]));
      }
      op[i] = r[k];
    }
  }
}

// ---------------------------------------------------------------- backward
// Blocks [0, chunks) sum one chunk of sorted entries each, one packet of columns per thread; the
// blocks after them write the zero rows of tokens that do not occur, kZeroTokens tokens each.
constexpr int kRowsAhead = 8;     // rows of a chunk whose loads are in flight together
constexpr int kZeroTokens = 64;

template <int DT, int VEC>
__global__ void __launch_bounds__(256)
embedding_bwd_kernel(const typename Elem<DT>::T* __restrict__ g, const int* __restrict__ start,
                     const int* __restrict__ pos, const int* __restrict__ tok, float* __restrict__ partial,
                     typename Elem<DT>::T* __restrict__ dtable, int chunks, int V, uint32_t packets, float scale) {
  pdl_enter();
  using E = Elem<DT>;
  using P = Pack<typename E::T, VEC>;
  const uint32_t c = blockIdx.y * blockDim.x + threadIdx.x;
  P* dp = reinterpret_cast<P*>(dtable);
  if ((int)blockIdx.x >= chunks) {
    const int v0 = ((int)blockIdx.x - chunks) * kZeroTokens;
    P zero;
#pragma unroll
    for (int e = 0; e < VEC; ++e) zero.v[e] = E::store(0.f);
    for (int v = v0; v < v0 + kZeroTokens && v < V; ++v)
      if (start[v] == start[v + 1] && c < packets) dp[(int64_t)v * packets + c] = zero;
    return;
  }
  const int chunk = blockIdx.x;
  const int i0 = chunk * kChunkRows, m = min(kChunkRows, start[V] - i0);   // the entries of this chunk
  if (m <= 0) return;
  __shared__ int s_pos[kChunkRows], s_tok[kChunkRows + 1];
  if (threadIdx.x < m) {
    s_pos[threadIdx.x] = pos[i0 + threadIdx.x];
    s_tok[threadIdx.x] = tok[i0 + threadIdx.x];
  }
  if (threadIdx.x == 0) s_tok[m] = -1;   // the chunk's end ends a run
  __syncthreads();
  if (c >= packets) return;
  const bool from_before = start[s_tok[0]] < i0, goes_on = start[s_tok[m - 1] + 1] > i0 + m;
  const P* gp = reinterpret_cast<const P*>(g);
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  bool first_run = true;
  for (int j0 = 0; j0 < m; j0 += kRowsAhead) {
    P r[kRowsAhead];
#pragma unroll
    for (int k = 0; k < kRowsAhead; ++k)
      if (j0 + k < m) r[k] = gp[(int64_t)s_pos[j0 + k] * packets + c];
#pragma unroll
    for (int k = 0; k < kRowsAhead; ++k) {
      const int j = j0 + k;
      if (j >= m) break;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += E::load(r[k].v[e]);
      if (s_tok[j + 1] == s_tok[j]) continue;
      // the run of s_tok[j] ends here (or goes on in the next chunk): a run that began in an earlier
      // chunk is that chunk's to finish (partial row 2 chunk), one that goes on is this chunk's
      // (partial row 2 chunk + 1)
      if ((first_run && from_before) || (j == m - 1 && goes_on)) {
        float* to = partial + ((int64_t)(2 * chunk + (first_run && from_before ? 0 : 1)) * packets + c) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) to[e] = acc[e];
      } else {
        P o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = E::store(scale * acc[e]);
        dp[(int64_t)s_tok[j] * packets + c] = o;
      }
      first_run = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    }
  }
}

// The rows of runs that cross chunks.  Block (chunk, y) finishes the run that begins in `chunk` and goes
// on past it, for 32 columns: its warps add contiguous shares of the run's partial rows, in order, then
// the warps' sums are added in warp order.
constexpr int kJoinWarps = 8;

template <int DT>
__global__ void __launch_bounds__(32 * kJoinWarps)
embedding_join_kernel(const int* __restrict__ start, const int* __restrict__ tok, const float* __restrict__ partial,
                      typename Elem<DT>::T* __restrict__ dtable, int V, int d, float scale) {
  pdl_enter();
  const int chunk = blockIdx.x, i0 = chunk * kChunkRows, i1 = i0 + kChunkRows;
  if (i1 >= start[V]) return;                       // no entries after this chunk
  const int t = tok[i1 - 1], s = start[t], e = start[t + 1];
  if (s < i0 || e <= i1) return;
  const int n = (e - 1) / kChunkRows - chunk + 1;   // partial rows: this chunk's, then one per later chunk
  const int col = blockIdx.y * 32 + threadIdx.x % 32, warp = threadIdx.x / 32;
  const int share = (n + kJoinWarps - 1) / kJoinWarps;
  const int k1 = min(n, (warp + 1) * share);
  float acc = 0.f;
  if (col < d)
#pragma unroll 8
    for (int k = warp * share; k < k1; ++k) acc += partial[(int64_t)(2 * (chunk + k) + (k == 0 ? 1 : 0)) * d + col];
  __shared__ float sum[kJoinWarps][32];
  sum[warp][threadIdx.x % 32] = acc;
  __syncthreads();
  if (warp == 0 && col < d) {
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) acc += sum[w][threadIdx.x];
    dtable[(int64_t)t * d + col] = Elem<DT>::store(scale * acc);
  }
}

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
  const int64_t items = n * (d / VEC);
  const int64_t per_block = 256 * kFwdItems;
  const dim3 grid((unsigned)std::min<int64_t>((items + per_block - 1) / per_block, 1 << 20));
  if (token_bits == 64)
    KRSI_CUDA_TRY(launch_pdl(embedding_fwd_kernel<DT, VEC, long long>, grid, dim3(256), 0, stream,
                             (const long long*)toks, (const T*)table, (T*)out, items, (uint32_t)(d / VEC), V, scale));
  else
    KRSI_CUDA_TRY(launch_pdl(embedding_fwd_kernel<DT, VEC, int>, grid, dim3(256), 0, stream, (const int*)toks,
                             (const T*)table, (T*)out, items, (uint32_t)(d / VEC), V, scale));
  return KRSI_OK;
}

struct BwdSpace {
  int *start, *pos, *tok;
  float* partial;
  size_t bytes;
};

inline BwdSpace bwd_space(void* base, int64_t n, int64_t V, int64_t d) {
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  char* p = static_cast<char*>(base);
  BwdSpace s;
  size_t off = 0;
  s.start = reinterpret_cast<int*>(p + off);
  off += up((size_t)(V + 1) * 4);
  s.pos = reinterpret_cast<int*>(p + off);
  off += up((size_t)n * 4);
  s.tok = reinterpret_cast<int*>(p + off);
  off += up((size_t)n * 4);
  s.partial = reinterpret_cast<float*>(p + off);
  off += up((size_t)tokens::chunks_of(n) * 2 * d * 4);
  s.bytes = off;
  return s;
}

template <int DT, int VEC>
int bwd(const void* g, const BwdSpace& s, void* dtable, int64_t n, int64_t V, int64_t d, float scale,
        cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const uint32_t packets = (uint32_t)(d / VEC);
  const int threads = (int)std::min<uint32_t>(256, std::max<uint32_t>(64, (packets + 31) / 32 * 32));
  const int chunks = (int)tokens::chunks_of(n);
  const dim3 grid((unsigned)(chunks + (V + kZeroTokens - 1) / kZeroTokens), (packets + threads - 1) / threads);
  KRSI_CUDA_TRY(launch_pdl(embedding_bwd_kernel<DT, VEC>, grid, dim3(threads), 0, stream, (const T*)g,
                           (const int*)s.start, (const int*)s.pos, (const int*)s.tok, s.partial, (T*)dtable, chunks,
                           (int)V, packets, scale));
  if (chunks > 1)
    KRSI_CUDA_TRY(launch_pdl(embedding_join_kernel<DT>, dim3(chunks - 1, (unsigned)((d + 31) / 32)),
                             dim3(32 * kJoinWarps), 0, stream, (const int*)s.start, (const int*)s.tok,
                             (const float*)s.partial, (T*)dtable, (int)V, (int)d, scale));
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
  *bytes = bwd_space(nullptr, n, V, d).bytes;
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
  const BwdSpace s = bwd_space(workspace, n, V, d);
  if (!workspace || workspace_bytes < s.bytes) return KRSI_ERR_WORKSPACE;
  if (!aligned16(workspace)) return KRSI_ERR_MISALIGNED;
  KRSI_CUDA_TRY(tokens::token_sort(toks, token_bits, n, V, padding_idx, s.start, s.pos, s.tok, stream));
  KRSI_EMB_DISPATCH(bwd, g, dtable, g, s, dtable, n, V, d, scale, stream)
}
