// token_rows.cuh - rows gathered and summed by token, shared by the embedding's gradient
// (embedding.cu) and the targets' part of the vocabulary projection's gradient (linear_ce.cu):
//   out[v] (+)= sum over the positions i with token v of weight[i] * g[i]
//
// The sum of the rows of one token has to be the same on every run, so it is taken in a fixed order: the
// positions are sorted by token first (token_sort), then cut into chunks of kChunkRows sorted entries,
// each summed by one block.  A token whose run lies inside one chunk is finished there;
// a run that crosses chunks leaves one partial row per chunk, which a second kernel adds in chunk order.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace krsi {
namespace tokens {

constexpr int kChunkRows = 16;

inline int64_t chunks_of(int64_t n) { return (n + kChunkRows - 1) / kChunkRows; }

// The order that tokens are sorted into: by their low bits (the groups), then by the rest.  Low ids are
// the frequent ones in most vocabularies; the groups spread them over the blocks of the sort.
struct Order {
  int bits;    // log2 of the groups
  int range;   // tokens per group
  __host__ __device__ __forceinline__ int key(int v) const { return (v & ((1 << bits) - 1)) * range + (v >> bits); }
  // One past the last key: 2^31 for the largest vocabularies, whose keys still fit an int.
  __host__ __device__ constexpr int64_t end() const { return (int64_t)range << bits; }
};
constexpr int kMaxRange = 512;
static_assert(Order{22, kMaxRange}.end() == (int64_t)1 << 31, "end() of the largest order");
inline Order order_of(int64_t V) {
  Order o{7, 0};   // 128 groups, more where a group would pass kMaxRange tokens
  while (((V - 1) >> o.bits) + 1 > kMaxRange) ++o.bits;
  o.range = (int)(((V - 1) >> o.bits) + 1);
  return o;
}

// The positions of tokens[0, n) sorted by token (in Order; equal tokens in an order that depends on n
// alone), those outside [0, V) and those equal to `skip` left out:
//   start[key(v)] .. start[key(v) + 1]   the sorted entries of token v (start[order.end()] = their number)
//   pos[i], tok[i]                       position and token of sorted entry i
// token_bits 32 or 64.  One kernel, no workspace beyond the outputs.
cudaError_t token_sort(const void* toks, int token_bits, int64_t n, int64_t V, int64_t skip, int* start, int* pos,
                       int* tok, cudaStream_t stream);

// Workspace of a sort and its partial rows (d columns), as offsets from one base.
struct Space {
  int *start, *pos, *tok;
  float* partial;
  Order order;
  size_t bytes;
};
inline Space space_at(void* base, int64_t n, int64_t V, int64_t d) {
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const uintptr_t p = reinterpret_cast<uintptr_t>(base);
  Space s;
  size_t off = 0;
  s.order = order_of(V);
  s.start = reinterpret_cast<int*>(p + off);
  off += up(((size_t)s.order.end() + 1) * 4);
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

// A thread's own packet from global to shared memory, asynchronously where the copy instruction exists
// for its width (4 bytes and more).  Only the thread that copied a packet reads it back, so waiting for
// its own copies is all the synchronisation there is.
template <typename P>
__device__ __forceinline__ void copy_packet(P* dst, const P* src) {
  if constexpr (sizeof(P) == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                 : "memory");
  else if constexpr (sizeof(P) >= 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                 "n"(sizeof(P))
                 : "memory");
  else
    *dst = *src;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The first blocks (if `chunks` is less than the grid) write the rows of tokens that do not occur,
// kZeroTokens tokens each; the last `chunks` blocks sum one chunk of sorted entries each, one packet of
// columns per thread.  A chunk's rows are staged in shared memory, all of its loads in flight at once: held
// in registers they cost so many that a third as much was in flight (measured at 32768 rows of 1152 16-bit
// values: 33 us against 39).
// Out: packet(v, c, sums, base) takes the VEC finished sums of token v's packet c with what fetch(v, first, c)
// read for it (a group's reads are in flight together), zero(v, c) an absent one, column(v, first, col, sum) one
// finished column.  first: the place of v's first entry among the sorted ones, a number below n that is v's own
// (kUsesFirst; else anything).
constexpr int kZeroTokens = 32;
constexpr int kGroupRows = 4;     // rows per group of copies

struct NoBase {};   // of an Out that reads nothing

template <int DT, int VEC, bool WEIGHTED, typename Out>
__global__ void __launch_bounds__(256)
sum_rows_kernel(const typename Elem<DT>::T* __restrict__ g, const float* __restrict__ weight,
                const int* __restrict__ start, const int* __restrict__ pos, const int* __restrict__ tok,
                float* __restrict__ partial, const Out out, const Order order, int n, int chunks, int V,
                uint32_t packets) {
  pdl_enter();
  using E = Elem<DT>;
  using P = Pack<typename E::T, VEC>;
  const uint32_t c = blockIdx.y * blockDim.x + threadIdx.x;
  const int chunk = (int)blockIdx.x - ((int)gridDim.x - chunks);
  if (chunk < 0) {
    const int v0 = (int)blockIdx.x * kZeroTokens, v = v0 + (int)(threadIdx.x % 32);
    const int k = v < V ? order.key(v) : 0;
    unsigned absent = __ballot_sync(0xffffffffu, v < V && start[k] == start[k + 1]);
    if (c < packets)
      for (; absent != 0; absent &= absent - 1) out.zero(v0 + __ffs(absent) - 1, c);
    return;
  }
  const int i0 = chunk * kChunkRows;
  __shared__ int s_pos[kChunkRows], s_tok[kChunkRows + 1], s_first[kChunkRows];
  __shared__ float s_weight[kChunkRows];
  // the chunk's entries, read beside the number that says how many of them there are
  const bool mine = threadIdx.x < kChunkRows && i0 + (int)threadIdx.x < n;
  const int p = mine ? pos[i0 + threadIdx.x] : 0, t = mine ? tok[i0 + threadIdx.x] : 0;
  const int m = min(kChunkRows, start[order.end()] - i0);
  if (m <= 0) return;
  if (threadIdx.x < m) {
    s_pos[threadIdx.x] = p;
    s_tok[threadIdx.x] = t;
    if (Out::kUsesFirst) s_first[threadIdx.x] = start[order.key(t)];
    if (WEIGHTED) s_weight[threadIdx.x] = weight[p];
  }
  if (threadIdx.x == 0) s_tok[m] = -1;   // the chunk's end ends a run
  __syncthreads();
  if (c >= packets) return;
  extern __shared__ __align__(16) unsigned char stage_raw[];
  P* stage = reinterpret_cast<P*>(stage_raw) + threadIdx.x;   // [kChunkRows][blockDim.x]
  const P* gp = reinterpret_cast<const P*>(g) + c;
#pragma unroll
  for (int j = 0; j < kChunkRows; ++j) {
    if (j < m) copy_packet(stage + j * blockDim.x, gp + (int64_t)s_pos[j] * packets);
    if (j % kGroupRows == kGroupRows - 1) copy_commit();
  }
  const bool from_before = start[order.key(s_tok[0])] < i0, goes_on = start[order.key(s_tok[m - 1]) + 1] > i0 + m;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  bool first_run = true;
  // a run that began in an earlier chunk is that chunk's to finish (partial row 2 chunk), one that goes on
  // in the next is this chunk's (partial row 2 chunk + 1)
  auto add_group = [&](int j0) {
    typename Out::Base base[kGroupRows];
#pragma unroll
    for (int k = 0; k < kGroupRows; ++k)
      if (j0 + k < m && s_tok[j0 + k + 1] != s_tok[j0 + k]) 
        base[k] = out.fetch(s_tok[j0 + k], Out::kUsesFirst ? s_first[j0 + k] : 0, c);
#pragma unroll
    for (int k = 0; k < kGroupRows; ++k) {
      const int j = j0 + k;
      if (j >= m) break;
      const P r = stage[j * blockDim.x];
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        acc[e] = WEIGHTED ? fmaf(s_weight[j], E::load(r.v[e]), acc[e]) : acc[e] + E::load(r.v[e]);
      if (s_tok[j + 1] == s_tok[j]) continue;
      if ((first_run && from_before) || (j == m - 1 && goes_on)) {
        float* to = partial + ((int64_t)(2 * chunk + (first_run && from_before ? 0 : 1)) * packets + c) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) to[e] = acc[e];
      } else {
        out.packet(s_tok[j], c, acc, base[k]);
      }
      first_run = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    }
  };
  static_assert(kChunkRows == 4 * kGroupRows, "four groups of copies");
  copy_wait<3>();
  add_group(0);
  copy_wait<2>();
  add_group(kGroupRows);
  copy_wait<1>();
  add_group(2 * kGroupRows);
  copy_wait<0>();
  add_group(3 * kGroupRows);
}

// The rows of runs that cross chunks, for 128 columns a block.  Each of the block's warps looks at one
// chunk: where a run begins in it and goes on past it, that run's partial rows (one per chunk) are added
// in chunk order.  Up to kShortRun of them the warp adds alone; a longer run is left to the whole block,
// whose warps add contiguous shares, in order, and then their sums in warp order.
constexpr int kJoinWarps = 8;
constexpr int kShortRun = 16;

template <typename Out>
__global__ void __launch_bounds__(32 * kJoinWarps)
join_rows_kernel(const int* __restrict__ start, const int* __restrict__ tok, const float* __restrict__ partial,
                 const Out out, const Order order, int d) {
  pdl_enter();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int col0 = blockIdx.y * 128 + lane;         // and 32, 64, 96 further
  // partial rows [k0, k1) of the run that begins in `chunk`: its tail, then the heads of later chunks
  auto add = [&](int chunk, int k0, int k1, float* acc) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = 0.f;
#pragma unroll 8
    for (int k = k0; k < k1; ++k) {
      const float* row = partial + (int64_t)(2 * (chunk + k) + (k == 0 ? 1 : 0)) * d;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col0 + 32 * j < d) acc[j] += row[col0 + 32 * j];
    }
  };
  auto put = [&](int t, const float* acc) {
    const int first = Out::kUsesFirst ? start[order.key(t)] : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col0 + 32 * j < d) out.column(t, first, col0 + 32 * j, acc[j]);
  };
  const int chunk = blockIdx.x * kJoinWarps + warp, i0 = chunk * kChunkRows, i1 = i0 + kChunkRows;
  int t = 0, n = 0;                                 // the run's token and partial rows; n = 0: none
  if (i1 < start[order.end()]) {
    t = tok[i1 - 1];
    const int k = order.key(t), e = start[k + 1];
    if (start[k] >= i0 && e > i1) n = (e - 1) / kChunkRows - chunk + 1;
  }
  float acc[4];
  if (n > 0 && n <= kShortRun) {
    add(chunk, 0, n, acc);
    put(t, acc);
  }
  __shared__ int s_n[kJoinWarps], s_t[kJoinWarps];
  __shared__ float sum[kJoinWarps][4][32];
  if (lane == 0) {
    s_n[warp] = n;
    s_t[warp] = t;
  }
  __syncthreads();
  for (int w = 0; w < kJoinWarps; ++w) {
    const int m = s_n[w];
    if (m <= kShortRun) continue;                   // the same for the whole block
    const int share = (m + kJoinWarps - 1) / kJoinWarps;
    add(blockIdx.x * kJoinWarps + w, min(m, warp * share), min(m, (warp + 1) * share), acc);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[warp][j][lane] = acc[j];
    __syncthreads();
    if (warp == 0) {
      for (int o = 1; o < kJoinWarps; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += sum[o][j][lane];
      put(s_t[w], acc);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- few positions
// Up to kFewRows positions need no sort: every block holds the whole token list, the block of a token's
// first position sums all of its rows, in position order, and the others end at once.  One launch in place
// of three; it costs n comparisons per block, and a long run is one block's work.
constexpr int kFewRows = 512;

// The tokens of [v0, v0 + 32) among tokens[0, n), as a mask (the same in every lane).
template <typename I>
__device__ __forceinline__ unsigned tokens_near(const I* tokens, int n, int v0) {
  unsigned mask = 0;
#pragma unroll 4
  for (int i = threadIdx.x % 32; i < n; i += 32) {
    const auto d = (std::make_unsigned_t<I>)tokens[i] - (std::make_unsigned_t<I>)v0;
    if (d < 32) mask |= 1u << (int)d;
  }
  return __reduce_or_sync(0xffffffffu, mask);
}

// The lane's token v0 + lane among tokens[0, n), n up to kFewRows: its first position, or -1.  Which lanes hold a
// lane's token follows from five ballots a step, one per bit of the difference (a loop over the hits cost the steps
// of 257 rows 5 us).
template <typename I>
__device__ __forceinline__ int first_near(const I* tokens, int n, int v0) {
  constexpr int kSteps = kFewRows / 32;
  const int lane = threadIdx.x % 32;
  unsigned d[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {   // all loads in flight together
    const int i = k * 32 + lane;
    const auto far = i < n ? (std::make_unsigned_t<I>)tokens[i] - (std::make_unsigned_t<I>)v0 : (std::make_unsigned_t<I>)32;
    d[k] = far < 32 ? (unsigned)far : 32u;
  }
  int first = -1;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    unsigned same = __ballot_sync(0xffffffffu, d[k] < 32);
    if (same == 0) continue;           // the same in every lane
#pragma unroll
    for (int b = 0; b < 5; ++b) {
      const unsigned set = __ballot_sync(0xffffffffu, d[k] >> b & 1);
      same &= lane >> b & 1 ? set : ~set;
    }
    if (same != 0 && first < 0) first = k * 32 + __ffs(same) - 1;
  }
  return first;
}

template <int DT, int VEC, bool WEIGHTED, typename Out, typename I>
__global__ void __launch_bounds__(256)
sum_few_kernel(const typename Elem<DT>::T* __restrict__ g, const float* __restrict__ weight,
               const I* __restrict__ toks, const Out out, int n, int V, int skip, uint32_t packets) {
  pdl_enter();
  using E = Elem<DT>;
  using P = Pack<typename E::T, VEC>;
  const uint32_t c = blockIdx.y * blockDim.x + threadIdx.x;
  const int i = (int)blockIdx.x - ((int)gridDim.x - n);   // the position whose token this block sums
  if (i < 0) {   // the first blocks (if any) write the rows of tokens that do not occur
    const int v0 = (int)blockIdx.x * kZeroTokens;
    unsigned present = tokens_near(toks, n, v0);
    if ((unsigned)(skip - v0) < 32u) present &= ~(1u << (skip - v0));
    for (int k = 0; k < kZeroTokens && v0 + k < V; ++k)
      if (!(present >> k & 1) && c < packets) out.zero(v0 + k, c);
    return;
  }
  __shared__ int s_rows[kFewRows], s_count;
  const I mine = toks[i];
  if (mine < 0 || mine >= (I)V || mine == (I)skip) return;
  if (threadIdx.x < 32) {
    int count = 0;
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + (int)threadIdx.x;
      const unsigned same = __ballot_sync(0xffffffffu, j < n && toks[j] == mine);
      if (same >> threadIdx.x & 1) s_rows[count + __popc(same & ((1u << threadIdx.x) - 1))] = j;
      count += __popc(same);
    }
    if (threadIdx.x == 0) s_count = count;
  }
  __syncthreads();
  if (s_rows[0] != i || c >= packets) return;   // an earlier position's block has this token
  const int m = s_count;
  extern __shared__ __align__(16) unsigned char stage_raw[];
  P* stage = reinterpret_cast<P*>(stage_raw) + threadIdx.x;   // [kChunkRows][blockDim.x]
  const P* gp = reinterpret_cast<const P*>(g) + c;
  const typename Out::Base base = out.fetch((int)mine, i, c);
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  for (int j0 = 0; j0 < m; j0 += kChunkRows) {
#pragma unroll 4
    for (int j = 0; j < kChunkRows && j0 + j < m; ++j)
      copy_packet(stage + j * blockDim.x, gp + (int64_t)s_rows[j0 + j] * packets);
    copy_commit();
    copy_wait<0>();
    for (int j = 0; j < kChunkRows && j0 + j < m; ++j) {
      const P r = stage[j * blockDim.x];
      const float w = WEIGHTED ? weight[s_rows[j0 + j]] : 1.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = WEIGHTED ? fmaf(w, E::load(r.v[e]), acc[e]) : acc[e] + E::load(r.v[e]);
    }
  }
  out.packet((int)mine, c, acc, base);
}

template <int DT, int VEC, bool WEIGHTED, typename Out, typename I>
cudaError_t sum_few(const void* g, const float* weight, const I* toks, const Out& out, bool zeros, int64_t n, int64_t V,
                    int64_t skip, int64_t d, cudaStream_t stream) {
  using T = typename Elem<DT>::T;
  const uint32_t packets = (uint32_t)(d / VEC);
  const int threads = (int)std::min<uint32_t>(256, std::max<uint32_t>(64, (packets + 31) / 32 * 32));
  const int64_t zero_blocks = zeros ? (V + kZeroTokens - 1) / kZeroTokens : 0;
  constexpr auto kern = sum_few_kernel<DT, VEC, WEIGHTED, Out, I>;
  const cudaError_t e = allow_smem<kern>(kChunkRows * 256 * 16);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3((unsigned)(zero_blocks + n), (packets + threads - 1) / threads), dim3(threads),
                    (size_t)kChunkRows * threads * VEC * sizeof(T), stream, (const T*)g, weight, toks, out, (int)n, (int)V,
                    (int)(skip >= 0 && skip < V ? skip : -1), packets);
}

// ---------------------------------------------------------------- many positions
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
  const size_t smem = (size_t)kChunkRows * threads * VEC * sizeof(T);   // at most 64 KB
  constexpr auto kern = sum_rows_kernel<DT, VEC, WEIGHTED, Out>;
  cudaError_t e = allow_smem<kern>(kChunkRows * 256 * 16);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kern, grid, dim3(threads), smem, stream, (const T*)g, weight, (const int*)s.start,
                 (const int*)s.pos, (const int*)s.tok, s.partial, out, s.order, (int)n, chunks, (int)V, packets);
  if (e != cudaSuccess || chunks == 1) return e;
  const dim3 join_grid((unsigned)((chunks - 1 + kJoinWarps - 1) / kJoinWarps), (unsigned)((d + 127) / 128));
  return launch_pdl(join_rows_kernel<Out>, join_grid, dim3(32 * kJoinWarps), 0, stream, (const int*)s.start,
                    (const int*)s.tok, (const float*)s.partial, out, s.order, (int)d);
}

}  // namespace tokens
}  // namespace krsi
