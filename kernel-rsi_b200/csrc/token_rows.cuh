// token_rows.cuh - rows gathered and summed by token, shared by the embedding's gradient
// (embedding.cu) and the targets' part of the vocabulary projection's gradient (linear_ce.cu):
//   out[v] (+)= sum over the positions i with token v of weight[i] * g[i]
//
// The sum of the rows of one token has to be the same on every run, so it is taken in position order:
// the positions are sorted by token first (token_sort, stable), then cut into chunks of kChunkRows
// sorted entries, each summed by one block.  A token whose run lies inside one chunk is finished there;
// a run that crosses chunks leaves one partial row per chunk, which a second kernel adds in chunk order.
#pragma once
#include <algorithm>

#include "common.cuh"

namespace krsi {
namespace tokens {

constexpr int kChunkRows = 32;

inline int64_t chunks_of(int64_t n) { return (n + kChunkRows - 1) / kChunkRows; }

// The positions of tokens[0, n) sorted by token (equal tokens in position order), those outside [0, V)
// and those equal to `skip` left out:
//   start[v] .. start[v + 1]   the sorted entries of token v (start[V] = their number)
//   pos[i], tok[i]             position and token of sorted entry i
// token_bits 32 or 64.  One kernel, no workspace beyond the outputs.
cudaError_t token_sort(const void* toks, int token_bits, int64_t n, int64_t V, int64_t skip, int* start, int* pos,
                       int* tok, cudaStream_t stream);

// Workspace of a sort and its partial rows (d columns), as offsets from one base.
struct Space {
  int *start, *pos, *tok;
  float* partial;
  size_t bytes;
};
inline Space space_at(void* base, int64_t n, int64_t V, int64_t d) {
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const uintptr_t p = reinterpret_cast<uintptr_t>(base);
  Space s;
  size_t off = 0;
  s.start = reinterpret_cast<int*>(p + off);
  off += up((size_t)(V + 1) * 4);
  s.pos = reinterpret_cast<int*>(p + off);
  off += up((size_t)n * 4);
  s.tok = reinterpret_cast<int*>(p + off);
  off += up((size_t)n * 4);
  s.partial = reinterpret_cast<float*>(p + off);
  off += up((size_t)chunks_of(n) * 2 * d * 4);
  s.bytes = off;
  return s;
}

// VEC elements moved as one access (16, 8, 4 or 2 bytes).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// Blocks [0, chunks) sum one chunk of sorted entries each, one packet of columns per thread; the blocks
// after them (if the grid has any) write the rows of tokens that do not occur, kZeroTokens tokens each.
// Out: packet(v, c, sums) takes the VEC finished sums of token v's packet c, zero(v, c) an absent one,
// column(v, col, sum) one finished column.
constexpr int kRowsAhead = 8;     // rows of a chunk whose loads are in flight together
constexpr int kZeroTokens = 64;

template <int DT, int VEC, bool WEIGHTED, typename Out>
__global__ void __launch_bounds__(256)
sum_rows_kernel(const typename Elem<DT>::T* __restrict__ g, const float* __restrict__ weight,
                const int* __restrict__ start, const int* __restrict__ pos, const int* __restrict__ tok,
                float* __restrict__ partial, const Out out, int chunks, int V, uint32_t packets) {
  pdl_enter();
  using E = Elem<DT>;
  using P = Pack<typename E::T, VEC>;
  const uint32_t c = blockIdx.y * blockDim.x + threadIdx.x;
  if ((int)blockIdx.x >= chunks) {
    const int v0 = ((int)blockIdx.x - chunks) * kZeroTokens;
    for (int v = v0; v < v0 + kZeroTokens && v < V; ++v)
      if (start[v] == start[v + 1] && c < packets) out.zero(v, c);
    return;
  }
  const int chunk = blockIdx.x;
  const int i0 = chunk * kChunkRows, m = min(kChunkRows, start[V] - i0);   // the entries of this chunk
  if (m <= 0) return;
  __shared__ int s_pos[kChunkRows], s_tok[kChunkRows + 1];
  __shared__ float s_weight[kChunkRows];
  if (threadIdx.x < m) {
    const int p = pos[i0 + threadIdx.x];
    s_pos[threadIdx.x] = p;
    s_tok[threadIdx.x] = tok[i0 + threadIdx.x];
    if (WEIGHTED) s_weight[threadIdx.x] = weight[p];
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
      for (int e = 0; e < VEC; ++e)
        acc[e] = WEIGHTED ? fmaf(s_weight[j], E::load(r[k].v[e]), acc[e]) : acc[e] + E::load(r[k].v[e]);
      if (s_tok[j + 1] == s_tok[j]) continue;
      // the run of s_tok[j] ends here (or goes on in the next chunk): a run that began in an earlier
      // chunk is that chunk's to finish (partial row 2 chunk), one that goes on is this chunk's
      // (partial row 2 chunk + 1)
      if ((first_run && from_before) || (j == m - 1 && goes_on)) {
        float* to = partial + ((int64_t)(2 * chunk + (first_run && from_before ? 0 : 1)) * packets + c) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) to[e] = acc[e];
      } else {
        out.packet(s_tok[j], c, acc);
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

template <typename Out>
__global__ void __launch_bounds__(32 * kJoinWarps)
join_rows_kernel(const int* __restrict__ start, const int* __restrict__ tok, const float* __restrict__ partial,
                 const Out out, int V, int d) {
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
    out.column(t, col, acc);
  }
}

// Both kernels over sorted positions `s` of n tokens; zeros: also write the rows of absent tokens.
template <int DT, int VEC, bool WEIGHTED, typename Out>
cudaError_t sum_by_token(const void* g, const float* weight, const Space& s, const Out& out, bool zeros, int64_t n,
                         int64_t V, int64_t d, cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const uint32_t packets = (uint32_t)(d / VEC);
  const int threads = (int)std::min<uint32_t>(256, std::max<uint32_t>(64, (packets + 31) / 32 * 32));
  const int chunks = (int)chunks_of(n);
  const int64_t zero_blocks = zeros ? (V + kZeroTokens - 1) / kZeroTokens : 0;
  const dim3 grid((unsigned)(chunks + zero_blocks), (packets + threads - 1) / threads);
  cudaError_t e = launch_pdl(sum_rows_kernel<DT, VEC, WEIGHTED, Out>, grid, dim3(threads), 0, stream, (const T*)g,
                             weight, (const int*)s.start, (const int*)s.pos, (const int*)s.tok, s.partial, out, chunks,
                             (int)V, packets);
  if (e != cudaSuccess || chunks == 1) return e;
  return launch_pdl(join_rows_kernel<Out>, dim3(chunks - 1, (unsigned)((d + 31) / 32)), dim3(32 * kJoinWarps), 0,
                    stream, (const int*)s.start, (const int*)s.tok, (const float*)s.partial, out, (int)V, (int)d);
}

}  // namespace tokens
}  // namespace krsi
