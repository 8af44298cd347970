// token_rows.cu - the positions of a token list sorted by token, in one kernel.
//
// Each block owns a group of the vocabulary (the tokens with the same low bits, at most kMaxRange) and
// reads all n tokens.  Reading everything 128 times sounds wasteful, but the tokens of a training batch
// are a few hundred KB that stay in L2, and it needs neither a second launch nor any exchange between
// blocks: a block counts the tokens of the groups before its own while it picks its own, and that count
// is where its entries begin.
//   1. pick: each warp goes through a share of the positions, 32 a step, and appends the block's tokens
//      to a list of its own in shared memory (a step without any costs about 20 instructions, and there
//      are n / 32 of them in every block: this is what bounds the kernel);
//   2. count: each warp counts its list by token, in counters of its own; the lanes of one step that hold
//      the same token are counted together;
//   3. an exclusive scan over (token, warp) turns the counters into offsets;
//   4. place: each warp walks its list again and writes the entries.
// Lists hold a tile of kTile positions; more positions take the steps tile by tile, and 1 again before 4.
// The order is fixed: by group, token, warp, tile and position.
// Measured at 32,768 tokens of a vocabulary of 32,768, ids as frequent as one over their rank: 12 us. (With
// contiguous ranges in place of the interleaved groups one block had half of the tokens: 41 us; with every
// step counted and ranked at once, without lists: 24 us.)
#include "token_rows.cuh"

namespace krsi {
namespace tokens {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 32768;
constexpr int kShare = kTile / kWarps;     // positions of a tile per warp
constexpr int kAhead = 8;                  // steps whose tokens are loaded together

template <typename T>
__global__ void __launch_bounds__(kThreads)
token_sort_kernel(const T* __restrict__ toks, int n, int V, int skip, const Order order, int share,
                  int* __restrict__ start, int* __restrict__ pos, int* __restrict__ tok) {
  pdl_enter();
  extern __shared__ int smem[];
  const int group = blockIdx.x, range = order.range, mask = (1 << order.bits) - 1;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int* cnt = smem;                                  // [kWarps][range]
  uint32_t* list = reinterpret_cast<uint32_t*>(smem + kWarps * range) + warp * share;   // bin << 16 | place in the tile's share
  int* mine = cnt + warp * range;
  __shared__ int warp_sum[kWarps];
  for (int i = threadIdx.x; i < kWarps * range; i += kThreads) cnt[i] = 0;

  int below = 0;
  // the block's tokens among positions [p0, p0 + share): appended to the list; returns their number
  auto pick = [&](int64_t p0) {
    int found = 0;
#pragma unroll 1
    for (int s = 0; s < share; s += 32 * kAhead) {
      T raw[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t p = p0 + s + k * 32 + lane;
        raw[k] = toks[p < n ? p : n - 1];
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int at = s + k * 32 + lane;
        const bool valid = raw[k] >= 0 && raw[k] < (T)V && raw[k] != (T)skip && at < share && p0 + at < n;
        const int v = valid ? (int)raw[k] : -1;     // (a -1's low bits are the last group's)
        const int g = v & mask;
        below += g < group;
        const bool hit = g == group && v >= 0;
        const unsigned in = __ballot_sync(0xffffffffu, hit);
        if (hit) list[found + __popc(in & ((1u << lane) - 1))] = (uint32_t)(v >> order.bits) << 16 | (uint32_t)at;
        found += __popc(in);
      }
    }
    __syncwarp();
    return found;
  };
  // calls f(live, entry, rank, count) for the list, a lane per entry: rank among the lanes of the step
  // with the same token, and their number
  auto walk = [&](int found, auto f) {
#pragma unroll 1
    for (int s = 0; s < found; s += 32) {
      const bool live = s + lane < found;
      const unsigned in = __ballot_sync(0xffffffffu, live);
      if (live) {
        const uint32_t entry = list[s + lane];
        const unsigned same = __match_any_sync(in, entry >> 16);
        f(in, entry, __popc(same & ((1u << lane) - 1)), __popc(same));
      }
      __syncwarp();
    }
  };

  __syncthreads();
  const int64_t tile = (int64_t)share * kWarps;
  int found = 0;
  for (int64_t p = 0; p < n; p += tile) {
    found = pick(p + (int64_t)warp * share);
    walk(found, [&](unsigned, uint32_t entry, int rank, int count) {
      if (rank == 0) mine[entry >> 16] += count;
    });
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
#pragma unroll 8
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
    if (group == mask && b == range - 1) start[order.end()] = first + total;
    if (total > 0) {
#pragma unroll 8
      for (int w = 0; w < kWarps; ++w) {
        const int c = cnt[w * range + b];
        cnt[w * range + b] = first;
        first += c;
      }
    }
  }
  __syncthreads();

  for (int64_t p = 0; p < n; p += tile) {
    const int64_t p0 = p + (int64_t)warp * share;
    if (tile < n) found = pick(p0);
    walk(found, [&](unsigned in, uint32_t entry, int rank, int count) {
      const int bin = entry >> 16, at = mine[bin] + rank;
      __syncwarp(in);
      if (rank == 0) mine[bin] = at + count;
      pos[at] = (int)p0 + (int)(entry & 0xffff);
      tok[at] = bin << order.bits | group;
    });
  }
}

template <typename T>
cudaError_t launch(const void* toks, int64_t n, int64_t V, int64_t skip, int* start, int* pos, int* tok,
                   cudaStream_t stream) {
  const Order order = order_of(V);
  const int64_t tile = n < kTile ? n : kTile;
  const int share = (int)((tile + 32 * kWarps - 1) / (32 * kWarps) * 32);
  const size_t smem = (size_t)kWarps * (order.range + share) * sizeof(int);
  static_assert(kWarps * (kMaxRange + kShare) * sizeof(int) <= 232448 - 1024, "shared memory budget");
  const cudaError_t e = allow_smem<token_sort_kernel<T>>((int)(kWarps * (kMaxRange + kShare) * sizeof(int)));
  if (e != cudaSuccess) return e;
  return launch_pdl(token_sort_kernel<T>, dim3(1u << order.bits), dim3(kThreads), smem, stream, (const T*)toks, (int)n,
                    (int)V, (int)skip, order, share, start, pos, tok);
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
