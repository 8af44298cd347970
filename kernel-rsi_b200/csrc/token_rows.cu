// token_rows.cu - a stable sort of token positions by token, in one kernel.
//
// Each block owns a range of the vocabulary (at most 1024 tokens) and reads all n tokens.  Reading
// everything 148 times sounds wasteful, but the tokens of a training batch are a few hundred KB that
// stay in L2, and it needs neither a second launch nor any exchange between blocks: a block counts the
// tokens below its range while it counts its own, and that count is where its entries begin.
//   1. each warp counts the in-range tokens of its contiguous share of the positions, in a row of
//      shared-memory counters of its own;
//   2. an exclusive scan over (token, warp) turns the counters into write offsets;
//   3. each warp walks its share again in order; the lanes of one step that hold the same token are
//      ranked by lane, so equal tokens land in position order.
// Bound by the L2 reads: two passes of n tokens per block.
#include "token_rows.cuh"

namespace krsi {
namespace tokens {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRange = 1024;
constexpr int kUnroll = 8;

template <typename T>
__global__ void __launch_bounds__(kThreads)
token_sort_kernel(const T* __restrict__ toks, int n, int V, int skip, int range, int* __restrict__ start,
                  int* __restrict__ pos, int* __restrict__ tok) {
  pdl_enter();
  extern __shared__ int cnt[];   // [kWarps][range]
  __shared__ int warp_sum[kWarps];
  const int lo = (int)blockIdx.x * range, hi = min(lo + range, V), bins = hi - lo;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i = threadIdx.x; i < kWarps * range; i += kThreads) cnt[i] = 0;
  __syncthreads();

  // this warp's positions [p0, p1): the step of one iteration is 32 * kUnroll
  const int share = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int64_t p0 = (int64_t)warp * share;
  const int p1 = (int)min((int64_t)n, p0 + share);
  int* mine = cnt + warp * range;
  // a token's bin: [0, bins) if owned, -1 if below the range, -2 if it counts nowhere here
  auto bin_of = [&](T t) { return t < 0 || t >= (T)V || t == (T)skip ? -2 : t < (T)lo ? -1 : t < (T)hi ? (int)t - lo : -2; };
  int below = 0;
  for (int64_t p = p0; p < p1; p += 32 * kUnroll) {
    T t[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) t[k] = p + k * 32 + lane < p1 ? toks[p + k * 32 + lane] : (T)-1;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int b = bin_of(t[k]);
      below += b == -1;
      if (b >= 0) atomicAdd(&mine[b], 1);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (lane == 0) warp_sum[warp] = below;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) base += warp_sum[w];
  __syncthreads();

  // exclusive scan over (token, warp): one token per thread
  const int b = threadIdx.x;
  int total = 0;
  if (b < bins)
    for (int w = 0; w < kWarps; ++w) total += cnt[w * range + b];
  int incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int first = base + incl - total;
  for (int w = 0; w < warp; ++w) first += warp_sum[w];
  if (b < bins) {
    start[lo + b] = first;
    if (lo + b == V - 1) start[V] = first + total;
    for (int w = 0; w < kWarps; ++w) {
      const int c = cnt[w * range + b];
      cnt[w * range + b] = first;
      first += c;
    }
  }
  __syncthreads();

  for (int64_t p = p0; p < p1; p += 32 * kUnroll) {
    T t[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) t[k] = p + k * 32 + lane < p1 ? toks[p + k * 32 + lane] : (T)-1;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int q = bin_of(t[k]);
      const unsigned in = __ballot_sync(0xffffffffu, q >= 0);
      if (in == 0) continue;
      if (q >= 0) {
        const unsigned same = __match_any_sync(in, q);
        const int rank = __popc(same & ((1u << lane) - 1)), at = mine[q] + rank;
        __syncwarp(in);
        if (rank == 0) mine[q] += __popc(same);
        pos[at] = (int)(p + k * 32 + lane);
        tok[at] = lo + q;
      }
      __syncwarp();
    }
  }
}

template <typename T>
cudaError_t launch(const void* toks, int64_t n, int64_t V, int64_t skip, int* start, int* pos, int* tok,
                   cudaStream_t stream) {
  const int sms = device_sm_count();
  const int64_t even = (V + sms - 1) / sms;
  const int range = (int)(even < kMaxRange ? even : kMaxRange);
  const size_t smem = (size_t)kWarps * range * sizeof(int);
  cudaError_t e = cudaFuncSetAttribute(token_sort_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)(kWarps * kMaxRange * sizeof(int)));
  if (e != cudaSuccess) return e;
  return launch_pdl(token_sort_kernel<T>, dim3((unsigned)((V + range - 1) / range)), dim3(kThreads), smem, stream,
                    (const T*)toks, (int)n, (int)V, (int)skip, range, start, pos, tok);
}

}  // namespace

cudaError_t token_sort(const void* toks, int token_bits, int64_t n, int64_t V, int64_t skip, int* start, int* pos,
                       int* tok, cudaStream_t stream) {
  if (skip < 0 || skip >= V) skip = -1;
  return token_bits == 64 ? launch<long long>(toks, n, V, skip, start, pos, tok, stream)
                          : launch<int>(toks, n, V, skip, start, pos, tok, stream);
}

}  // namespace tokens
}  // namespace krsi
