// token_rows.cu - a stable sort of token positions by token, in one kernel.
//
// Each block owns a group of the vocabulary (the tokens with the same low bits, at most 1024) and reads
// all n tokens.  Reading everything 128 times sounds wasteful, but the tokens of a training batch are a
// few hundred KB that stay in L2, and it needs neither a second launch nor any exchange between blocks: a
// block counts the tokens of the groups before its own while it counts its own, and that count is where
// its entries begin.
//   1. each warp counts its block's tokens in a contiguous share of the positions, in a row of
//      shared-memory counters of its own;
//   2. an exclusive scan over (token, warp) turns the counters into write offsets;
//   3. each warp walks its share again in order; the lanes of one step that hold the same token are
//      ranked by lane, so equal tokens land in position order.
// Up to kHeld * 1024 tokens a lane holds its share in registers between 1 and 3, with all its loads in
// flight together; above, the tokens are read again.  Measured at 32,768 tokens: SORT_HELD against SORT_LOOP.
#include "token_rows.cuh"

namespace krsi {
namespace tokens {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kHeld = 32;     // tokens a lane holds
constexpr int kAhead = 8;     // loads in flight where they are not held

// A lane's token in one step of its warp: its bin, its rank among the lanes with the same bin, and their
// number, packed; negative: not in this block's range.
__device__ __forceinline__ int entry_of(int bin, unsigned lane) {
  const unsigned in = __ballot_sync(0xffffffffu, bin >= 0);
  if (in == 0 || bin < 0) return -1;
  const unsigned same = __match_any_sync(in, bin);
  return bin | __popc(same & ((1u << lane) - 1)) << 10 | __popc(same) << 16;
}
__device__ __forceinline__ int bin_of(int entry) { return entry & 1023; }
__device__ __forceinline__ int rank_of(int entry) { return entry >> 10 & 31; }
__device__ __forceinline__ int count_of(int entry) { return entry >> 16; }

template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads)
token_sort_kernel(const T* __restrict__ toks, int n, int V, int skip, const Order order, int* __restrict__ start,
                  int* __restrict__ pos, int* __restrict__ tok) {
  pdl_enter();
  extern __shared__ int cnt[];   // [kWarps][range]
  __shared__ int warp_sum[kWarps];
  const int group = blockIdx.x, range = order.range, mask = (1 << order.bits) - 1;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  // this warp's positions [p0, p1), 32 a step
  const int share = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int64_t p0 = (int64_t)warp * share;
  const int p1 = (int)min((int64_t)n, p0 + share);
  int* mine = cnt + warp * range;
  int below = 0;
  // the token's bin in the group, or -1; counts it if it belongs to a group before
  auto classify = [&](T t) {
    if (t < 0 || t >= (T)V || t == (T)skip) return -1;
    const int v = (int)t, g = v & mask;
    below += g < group;
    return g == group ? v >> order.bits : -1;
  };
  auto load = [&](int64_t p) { return p + lane < p1 ? toks[p + lane] : (T)-1; };
  auto count = [&](int entry) {
    if (entry >= 0 && rank_of(entry) == 0) mine[bin_of(entry)] += count_of(entry);
    __syncwarp();
  };
  auto place = [&](int entry, int64_t p) {
    const int at = entry >= 0 ? mine[bin_of(entry)] + rank_of(entry) : 0;
    __syncwarp();
    if (entry >= 0) {
      if (rank_of(entry) == 0) mine[bin_of(entry)] += count_of(entry);
      pos[at] = (int)(p + lane);
      tok[at] = bin_of(entry) << order.bits | group;
    }
    __syncwarp();
  };

  T held[HELD ? kHeld : 1];
  int entry[HELD ? kHeld : 1];
  if (HELD) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) held[k] = load(p0 + k * 32);
  }
  for (int i = threadIdx.x; i < kWarps * range; i += kThreads) cnt[i] = 0;
  __syncthreads();
  if (HELD) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      entry[k] = -1;
      if (p0 + k * 32 < p1) {
        entry[k] = entry_of(classify(held[k]), lane);
        if (__any_sync(0xffffffffu, entry[k] >= 0)) count(entry[k]);
      }
    }
  } else {
    for (int64_t p = p0; p < p1; p += 32 * kAhead) {
      T t[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) t[k] = load(p + k * 32);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int e = entry_of(classify(t[k]), lane);
        if (__any_sync(0xffffffffu, e >= 0)) count(e);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (lane == 0) warp_sum[warp] = below;
  __syncthreads();
  int base = warp_sum[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o);
  __syncthreads();

  // exclusive scan over (token, warp): one token per thread
  const int b = threadIdx.x;
  int total = 0;
  if (b < range) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += cnt[w * range + b];
  }
  int incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int before = lane < warp ? warp_sum[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  int first = base + before + incl - total;
  if (b < range) {
    start[group * range + b] = first;
    if (group == mask && b == range - 1) start[(group + 1) * range] = first + total;
    if (total > 0) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int c = cnt[w * range + b];
        cnt[w * range + b] = first;
        first += c;
      }
    }
  }
  __syncthreads();

  if (HELD) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (__any_sync(0xffffffffu, entry[k] >= 0)) place(entry[k], p0 + k * 32);
  } else {
    for (int64_t p = p0; p < p1; p += 32 * kAhead) {
      T t[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) t[k] = load(p + k * 32);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int e = entry_of(classify(t[k]), lane);
        if (__any_sync(0xffffffffu, e >= 0)) place(e, p + k * 32);
      }
    }
  }
}

template <typename T>
cudaError_t launch(const void* toks, int64_t n, int64_t V, int64_t skip, int* start, int* pos, int* tok,
                   cudaStream_t stream) {
  const Order order = order_of(V);
  const size_t smem = (size_t)kWarps * order.range * sizeof(int);
  auto kern = n <= (int64_t)kHeld * 32 * kWarps ? token_sort_kernel<T, true> : token_sort_kernel<T, false>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)(kWarps * kMaxRange * sizeof(int)));
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(1u << order.bits), dim3(kThreads), smem, stream, (const T*)toks, (int)n, (int)V,
                    (int)skip, order, start, pos, tok);
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
